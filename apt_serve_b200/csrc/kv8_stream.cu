// Up to 16 query rows per request over the 8-bit cache (kv8_common.cuh): decode, drafted tokens.  fp16 / bf16 queries, head sizes 64, 128.
//
// HBM-bound: the codes are read once, 2 D bytes a token and head.  One CTA of a single warp per (request, part of the tokens, head), the
// heads next to one another, so that a token's row is read by warps that run at the same time; a group of 16 tokens (which never
// straddles a block) at a time, asynchronous copies bring the next ones to shared memory.
// Both products are taken the other way round, the cache's rows as the 16-row operand A of mma.sync.m16n8k16 and the query rows as the
// 8 columns of B.  A's fragments are what plain vector loads of the rows give, if the dimensions are counted in another order (a sum over
// them does not mind, and the output's are written where they belong); lane (g, j) = (lane / 4, lane % 4):
//   S^T = K Q^T   A (16 tokens x 16 dims): four codes of token g and of token g + 8 at a time, of the lane's 16 consecutive dims
//                 16 j ... 16 j + 15 of a 64-byte half row; B holds the query's elements in the same order
//   O^T += V^T P^T  A (16 dims x 16 tokens): tokens 2 j, 2 j + 1, 2 j + 8, 2 j + 9 of the lane's D / 8 consecutive dims, the tokens
//                 paired by a byte permutation; tile i has dims (D / 8) g + 2 i and + 1 in rows g and g + 8.  P^T comes from S^T's
//                 layout by a transposition in registers (movmatrix)
// Every e4m3 number is an fp16 number.  The scales, the weights' two references and their one fp16 term are those of the tile kernel
// (kv8_prefix.cu).
// Measured on one B200: one row of 256 OPT-13B requests (2.69 GB) 501 us back to back, 82 % of the measured copy rate.  What bounds it is
// half memory and half the warps' own instructions (about 210 a group of 16 tokens: 64 conversions and 16 permutations, 16 products, 50
// for the softmax).  Before this form: registers as the only staging 904 us, a ring of asynchronous copies 573, the query rows as the
// 16-row operand (twice the products) 590.
#include "kv8_common.cuh"

#include <type_traits>

namespace aps {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr float kSlack = 8.f;   // log2 of how much the weights' reference may have grown before O is rescaled
constexpr float kUp = 7.f;      // log2 of what the weights are kept at

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {   // of an 8 x 8 matrix of 16-bit elements
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 16 (or 4) bytes to shared memory; of which none: zeros.
__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool some) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(some ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }
__device__ __forceinline__ uint4 shared16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ uint2 shared8(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
  return v;
}
__device__ __forceinline__ float2 shared_pair(uint32_t at) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at));
  return v;
}
// Where piece c (16 bytes) of a row of D bytes lies in a group's 16 rows: 8 lanes' loads, of two tokens' pieces (K) or of four tokens'
// (V), meet different banks (V at D = 64: two lanes each).
template <int D> __device__ __forceinline__ uint32_t piece_at(int row, int c) {
  if constexpr (D == 128) return (uint32_t)(row * 128 + ((c ^ (row & 7) ^ ((row & 1) << 2)) << 4));
  else return (uint32_t)(row * 64 + ((c ^ (row >> 1 & 3)) << 4));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Groups of 16 tokens of a part, at least.  A group takes a warp a quarter of a microsecond, joining the parts four or five, so that
// tables of up to 16 groups are not cut and parts have eight at least.  Where parts of up to 40 fill the GPU once, as many as fill it
// (a 30 011-token OPT-1.3B context: 26 groups 34 us, 16 37, 48 41); else 16, and 32 where there are many of them (128 OPT-66B tp 8
// requests: 16 groups 69 us, 32 77; 256 OPT-13B requests 519 and 500).
int64_t units_at_once() { return (int64_t)sm_count() * 16; }   // warps on the GPU at a time (the kernel of 9 - 16 rows: 10 an SM, not planned for)
int part_groups(const Kv8Call& c) {
  const int64_t gpu = units_at_once();
  const int64_t each = (int64_t)c.max_blocks * c.cache.block_size / 16, units = (int64_t)c.batch * c.cache.heads;
  if (each <= 16) return 16;
  if (units < gpu) {
    const int64_t parts = gpu / units, n = (each + parts - 1) / parts;
    if (n <= 40) return (int)(n < 8 ? 8 : n);
  }
  return each * units < 128 * gpu ? 16 : 32;
}

template <int D> __host__ __device__ constexpr int stages() { return D == 128 ? 3 : 6; }   // groups of a warp in shared memory
template <int D> __host__ __device__ constexpr int stage_bytes() { return 2 * 16 * D + 16; }

// kRows: query rows at most, 1, 8 or 16.
template <typename T, int D, int kRows>
__global__ void __launch_bounds__(32, kRows == 16 ? 10 : 16)
kv8_stream_kernel(const Kv8Call c, const Kv8Parts parts, const int part_groups, const uint32_t blocks_magic, const int vec) {
  constexpr int kCols = D / 64, kPer = D / 8, kStages = stages<D>();   // 64-byte pieces of a row; dims of a lane in V
  constexpr int kSets = kRows == 16 ? 2 : 1, kEach = kRows == 1 ? 1 : 2;   // sets of 8 query rows; rows of a set whose softmax a lane keeps
  extern __shared__ __align__(128) uint8_t ring_raw[];
  const int lane = threadIdx.x, g = lane >> 2, j = lane & 3;
  chain_wait();
  chain_next();
  const int head = blockIdx.x % c.cache.heads, part = blockIdx.x / c.cache.heads, req = part / parts.splits, split = part % parts.splits;
  if (blockIdx.x == 0 && threadIdx.x == 0) parts.plan[kPlanStatus] = kStatusOk;
  const int start = c.starts != nullptr ? c.starts[req] : req;
  const int rows_all = c.starts != nullptr ? c.starts[req + 1] - start : 1, n_rows = min(c.starts != nullptr ? min(kRows, c.max_rows) : 1, rows_all);
  if (n_rows <= 0) return;
  const int bs = c.cache.block_size, ctx = max(0, min(c.seq_lens[req], c.max_blocks * bs));
  const int first = ctx - rows_all;                    // own position of the first row
  const int all = (ctx + 15) / 16, per = max(part_groups, (all + parts.splits - 1) / parts.splits);   // groups of 16 tokens
  const int group0 = min(all, split * per), n_groups = min(all, group0 + per) - group0;
  const int32_t* table = c.tables + (int64_t)req * c.max_blocks;
  const int64_t row_bytes = (int64_t)c.cache.heads * D;
  const uint32_t per_block = (uint32_t)bs / 16, ring = (uint32_t)__cvta_generic_to_shared(ring_raw);
  auto block_at = [&](uint32_t group) { return blocks_magic ? __umulhi(group, blocks_magic) : group; };   // group / per_block
  auto block_of = [&](int k) { return k < n_groups ? table[block_at(group0 + k)] : -1; };
  // group k on its way to stage k % kStages
  constexpr int kPieces = D / 16, kAtOnce = 32 / kPieces, kCopies = 16 / kAtOnce;
  const int piece = lane % kPieces, r0 = lane / kPieces;
  const int64_t column = (int64_t)head * D + piece * 16 + r0 * row_bytes, step = kAtOnce * row_bytes;
  const uint8_t *keys = c.cache.key + column, *values = c.cache.value + column;
  const float* scales = (lane == 0 ? c.cache.key_scale : c.cache.value_scale) + head;
  auto fetch = [&](int k, int block) {
    const uint32_t group = group0 + k, to = ring + k % kStages * stage_bytes<D>();
    const bool in = block >= 0 && block < c.cache.num_blocks;
    if (!in) block = 0;   // something that can be read
    const int64_t from = block * c.cache.block_stride + (int64_t)((group - block_at(group) * per_block) * 16) * row_bytes;
    const uint8_t *kp = keys + from, *vp = values + from;
    const int live = in ? ctx - (int)group * 16 : 0;   // tokens that count
    if (live >= 16) {
#pragma unroll
      for (int i = 0; i < kCopies; ++i) copy16(to + piece_at<D>(r0 + i * kAtOnce, piece), kp + i * step);
#pragma unroll
      for (int i = 0; i < kCopies; ++i) copy16(to + 16 * D + piece_at<D>(r0 + i * kAtOnce, piece), vp + i * step);
    } else {              // rows behind the last token: zeros, whatever they hold
#pragma unroll
      for (int i = 0; i < kCopies; ++i) copy16(to + piece_at<D>(r0 + i * kAtOnce, piece), kp + i * step, r0 + i * kAtOnce < live);
#pragma unroll
      for (int i = 0; i < kCopies; ++i) copy16(to + 16 * D + piece_at<D>(r0 + i * kAtOnce, piece), vp + i * step, r0 + i * kAtOnce < live);
    }
    if (lane < 2) {
      const uint32_t at = to + 2 * 16 * D + 4 * lane;
      if (in) copy4(at, scales + block * c.cache.scale_stride);
      else asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(lane == 0 ? __int_as_float(0x7fc00000) : 0.f) : "memory");   // NaN scores
    }
  };
  int next = block_of(0);
#pragma unroll
  for (int k = 0; k < kStages - 1; ++k) {
    if (k < n_groups) fetch(k, next);
    copy_commit();
    next = block_of(k + 1);
  }

  // the query's fragments, row g (and g + 8): a half row's 16 dims of the lane, four at a time; bf16 as fp16 times a power of two per row
  uint32_t qb[kSets][D / 16][2];
  float coef[kSets][kEach];
#pragma unroll
  for (int q = 0; q < kSets; ++q) {
    const int row = g + 8 * q;
    const int64_t t = (int64_t)start + row;
    const bool mine = row < n_rows && t >= 0 && t < c.rows;
    const T* src = static_cast<const T*>(c.query) + (mine ? t : 0) * c.query_stride + (int64_t)head * D + j * 16;
    float x[16 * kCols], top = 0.f;
#pragma unroll
    for (int h = 0; h < kCols; ++h) {
      if (mine && vec) {
        Vec16<T>::unpack(*reinterpret_cast<const uint4*>(src + 64 * h), x + 16 * h);
        Vec16<T>::unpack(*reinterpret_cast<const uint4*>(src + 64 * h + 8), x + 16 * h + 8);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) x[16 * h + e] = mine ? Elem<T>::to_float(src[64 * h + e]) : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (fabsf(x[16 * h + e]) <= 3.402823466e38f) top = fmaxf(top, fabsf(x[16 * h + e]));
    }
    float down = 1.f, up = 1.f;
    if (std::is_same<T, __nv_bfloat16>::value) {
      top = fmaxf(top, __shfl_xor_sync(kFull, top, 1));
      top = fmaxf(top, __shfl_xor_sync(kFull, top, 2));
      const int p = min(120, 127 + 14 - (int)(__float_as_uint(top) >> 23));   // the largest element to 2^14 ... 2^15
      down = __uint_as_float((uint32_t)(127 + p) << 23);
      up = __uint_as_float((uint32_t)(127 - p) << 23);
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) coef[q][e] = parts.scale_log2 * __shfl_sync(kFull, up, kRows == 1 ? 0 : (2 * j + e) * 4);   // of row 2 j + e
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      qb[q][s][0] = half2_bits(x[4 * s] * down, x[4 * s + 1] * down);
      qb[q][s][1] = half2_bits(x[4 * s + 2] * down, x[4 * s + 3] * down);
    }
  }

  const bool both = kSets == 2 && n_rows > 8;   // most requests of a batch can have fewer rows than the largest
  // columns 2 j, 2 j + 1 of a set are the lane's query rows
  float acc[kSets][D / 16][4];   // dims' rows g, g, g + 8, g + 8
#pragma unroll
  for (int q = 0; q < kSets; ++q)
#pragma unroll
    for (int i = 0; i < D / 16; ++i) acc[q][i][0] = acc[q][i][1] = acc[q][i][2] = acc[q][i][3] = 0.f;
  float m[kSets][kEach], l[kSets][kEach], ref[kSets][kEach];
#pragma unroll
  for (int q = 0; q < kSets; ++q)
#pragma unroll
    for (int e = 0; e < kEach; ++e) { m[q][e] = ref[q][e] = -INFINITY; l[q][e] = 0.f; }

  auto consume = [&](int k) {
    const int t0 = (group0 + k) * 16;
    const uint32_t at = ring + k % kStages * stage_bytes<D>();
    const float2 scale = shared_pair(at + 2 * 16 * D);
    float s[kSets][4];   // tokens g, g, g + 8, g + 8
#pragma unroll
    for (int q = 0; q < kSets; ++q) s[q][0] = s[q][1] = s[q][2] = s[q][3] = 0.f;
#pragma unroll
    for (int h = 0; h < kCols; ++h) {
      const uint4 lo = shared16(at + piece_at<D>(g, 4 * h + j)), hi = shared16(at + piece_at<D>(g + 8, 4 * h + j));
      const uint32_t w[2][4] = {{lo.x, lo.y, lo.z, lo.w}, {hi.x, hi.y, hi.z, hi.w}};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t a0, a1, a2, a3;
        e4m3x4_to_f16x4(w[0][e], a0, a2);
        e4m3x4_to_f16x4(w[1][e], a1, a3);
#pragma unroll
        for (int q = 0; q < kSets; ++q)
          if (q == 0 || both) mma16816(s[q], a0, a1, a2, a3, qb[q][4 * h + e][0], qb[q][4 * h + e][1]);
      }
    }
    const float lv = lg2(scale.y);
    uint32_t p[kSets][2];   // P^T's fragments
    const bool edge = t0 + 15 > first;   // some row does not attend to all of the tokens
    bool any = false;
    float down[kSets][2];
#pragma unroll
    for (int q = 0; q < kSets; ++q) {
      float w[2][2] = {{0.f, 0.f}, {0.f, 0.f}};   // [tokens g, g + 8][rows]
      down[q][0] = down[q][1] = 1.f;
      p[q][0] = p[q][1] = 0u;
      if (q == 1 && !both) continue;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        float by = coef[q][e] * scale.x, x0 = s[q][e], x1 = s[q][2 + e];
        if (edge) {
          // -infinity times a factor that is 0 or NaN would be NaN: such a factor goes into the scores
          const int seen = first + (kRows == 1 ? 0 : 8 * q + 2 * j + e) - t0;   // the last token that the row attends to
          const bool plain = by > 0.f;
          const float fill = by == 0.f ? 0.f : __int_as_float(0x7fc00000);
          if (!plain) by = 1.f;
          x0 = g > seen ? -INFINITY : plain ? x0 : fill;
          x1 = g + 8 > seen ? -INFINITY : plain ? x1 : fill;
        }
        float top = fmaxf(x0, x1);
        top = fmaxf(top, __shfl_xor_sync(kFull, top, 4));
        top = fmaxf(top, __shfl_xor_sync(kFull, top, 8));
        top = fmaxf(top, __shfl_xor_sync(kFull, top, 16)) * by;   // NaN counts as none
        const float m_new = fmaxf(m[q][e], top), r_new = fmaxf(-INFINITY, top + lv);
        const bool move = r_new > ref[q][e] && !(r_new - ref[q][e] <= kSlack);
        any = any || move;
        down[q][e] = move && ref[q][e] != -INFINITY ? ex2(ref[q][e] - r_new) : 1.f;
        if (move) ref[q][e] = r_new;
        const float shift = m_new == -INFINITY ? 0.f : m_new, base = shift - (ref[q][e] == -INFINITY ? 0.f : ref[q][e]) + kUp + lv;
        const float off = base < -60.f ? -60.f : base, from = off - shift;
        w[0][e] = ex2(fmaf(x0, by, from));
        w[1][e] = ex2(fmaf(x1, by, from));
        l[q][e] = fmaf(w[0][e] + w[1][e], ex2(-off), m[q][e] == -INFINITY ? 0.f : l[q][e] * ex2(m[q][e] - shift));
        m[q][e] = m_new;
      }
      p[q][0] = transposed(half2_bits(w[0][0], w[0][1]));
      p[q][1] = transposed(half2_bits(w[1][0], w[1][1]));
    }
    if (__any_sync(kFull, any)) {
#pragma unroll
      for (int q = 0; q < kSets; ++q)
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[q][i][e] *= down[q][e & 1];
    }
    uint32_t v[4][kPer / 4];   // tokens 2 j, 2 j + 1, 2 j + 8, 2 j + 9
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int row = 2 * j + (t & 1) + 8 * (t >> 1);
      if constexpr (D == 128) {
        const uint4 x = shared16(at + 16 * D + piece_at<D>(row, g));
        v[t][0] = x.x; v[t][1] = x.y; v[t][2] = x.z; v[t][3] = x.w;
      } else {
        const uint2 x = shared8(at + 16 * D + piece_at<D>(row, g >> 1) + 8 * (g & 1));
        v[t][0] = x.x; v[t][1] = x.y;
      }
    }
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {   // dims 2 i and 2 i + 1 of the lane's
      const uint32_t b0 = __byte_perm(v[0][i / 2], v[1][i / 2], i & 1 ? 0x7362 : 0x5140);
      const uint32_t b1 = __byte_perm(v[2][i / 2], v[3][i / 2], i & 1 ? 0x7362 : 0x5140);
      uint32_t a0, a1, a2, a3;
      e4m3x4_to_f16x4(b0, a0, a1);
      e4m3x4_to_f16x4(b1, a2, a3);
#pragma unroll
      for (int q = 0; q < kSets; ++q)
        if (q == 0 || both) mma16816(acc[q][i], a0, a1, a2, a3, p[q][0], p[q][1]);
    }
  };
  for (int k = 0; k < n_groups; ++k) {
    copy_wait<kStages - 2>();
    __syncwarp();   // every lane's copies of group k are there, every lane has read group k - 1
    if (k + kStages - 1 < n_groups) fetch(k + kStages - 1, next);
    copy_commit();
    next = block_of(k + kStages);
    consume(k);
  }
  copy_wait<0>();

  // the rows: the lane has dims kPer g ... kPer g + kPer - 1 of its query rows
#pragma unroll
  for (int q = 0; q < kSets; ++q)
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int row = 8 * q + 2 * j + e;
      const int64_t t = (int64_t)start + row;
      float sum = l[q][e];
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(kFull, sum, o);
      if (row >= n_rows || t < 0 || t >= c.rows) continue;
      // relative to 2^m, in two steps: with the least scales the factor is 2^-133, below the normal range
      const float root = ref[q][e] == -INFINITY ? 0.f : ex2(0.5f * (ref[q][e] - kUp - (m[q][e] == -INFINITY ? 0.f : m[q][e])));
      float by = root;
      if (parts.splits == 1) by /= sum;    // nothing but scores of -infinity: NaN
      const bool none = first + row < 0;   // a row before the first token
      const int64_t unit = (t * c.cache.heads + head) * parts.splits + split;
      float x[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) x[i] = none ? 0.f : acc[q][i / 2][2 * (i & 1) + e] * root * by;
      if (parts.splits > 1) {
        float* dst = parts.acc + unit * D + kPer * g;
#pragma unroll
        for (int i = 0; i < kPer; i += 4) *reinterpret_cast<float4*>(dst + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
        if (g == 0) parts.ml[unit] = make_float2(m[q][e], sum);
      } else {
        T* dst = static_cast<T*>(c.out) + t * c.out_stride + (int64_t)head * D + kPer * g;
        if (vec) {
          struct alignas(16) Eight { T x[8]; };
#pragma unroll
          for (int i = 0; i < kPer; i += 8) {
            Eight o;
#pragma unroll
            for (int d = 0; d < 8; ++d) o.x[d] = Elem<T>::from_float(x[i + d]);
            *reinterpret_cast<Eight*>(dst + i) = o;
          }
        } else {
#pragma unroll
          for (int i = 0; i < kPer; ++i) dst[i] = Elem<T>::from_float(x[i]);
        }
      }
    }
}

template <typename T, int D, int kRows>
int launch(const Kv8Call& c, const Kv8Parts& parts, cudaStream_t stream) {
  static bool done[64] = {false};
  auto kernel = kv8_stream_kernel<T, D, kRows>;
  constexpr int smem = stages<D>() * stage_bytes<D>();
  int dev = 0;
  APS_CUDA(cudaGetDevice(&dev));
  APS_REQUIRE(dev >= 0 && dev < 64, APS_ERR_CUDA, "device index %d out of range", dev);
  if (!done[dev]) {
    APS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    APS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    done[dev] = true;
  }
  const int64_t grid = (int64_t)c.batch * parts.splits * c.cache.heads;
  APS_REQUIRE(grid < (int64_t(1) << 31), APS_ERR_SHAPE, "kv8_attention: too many requests");
  const int vec = aligned_to(c.query, 16) && aligned_to(c.out, 16) && c.query_stride % 8 == 0 && c.out_stride % 8 == 0;
  return launch_chained("kv8_stream_kernel", kernel, (unsigned)grid, 32, smem, stream, c, parts, part_groups(c),
                        kv8_blocks_magic(c.cache.block_size), vec);
}

template <typename T, int D>
int launch_rows(const Kv8Call& c, const Kv8Parts& parts, cudaStream_t stream) {
  if (c.starts == nullptr || c.max_rows == 1) return launch<T, D, 1>(c, parts, stream);
  return c.max_rows <= 8 ? launch<T, D, 8>(c, parts, stream) : launch<T, D, 16>(c, parts, stream);
}

template <typename T>
int launch_typed(const Kv8Call& c, const Kv8Parts& parts, cudaStream_t stream) {
  return c.cache.head_size == 128 ? launch_rows<T, 128>(c, parts, stream) : launch_rows<T, 64>(c, parts, stream);
}

}  // namespace

bool kv8_stream_takes(const Kv8Call& c) {
  return (c.starts == nullptr || c.max_rows <= 16) && (c.dtype == APS_F16 || c.dtype == APS_BF16) &&
         (c.cache.head_size == 64 || c.cache.head_size == 128) && c.cache.num_blocks > 0 && c.scale >= 1.17549435e-38f && c.scale < 1.70141183e38f;
}

// Parts that a request's tokens are cut into.
int kv8_stream_splits(const Kv8Call& c) {
  const int64_t groups = (int64_t)c.max_blocks * c.cache.block_size / 16, n = (groups + part_groups(c) - 1) / part_groups(c);
  // with many units and wide tables (of which the lengths may use little) no more than a few
  const int64_t units = (int64_t)c.batch * c.cache.heads, most = (units_at_once() * 4 + units - 1) / units;
  const int64_t some = n < most ? n : most < 4 ? (n < 4 ? n : 4) : most;
  return (int)(some > 1024 ? 1024 : some);   // as many as the joining kernel takes
}

int launch_kv8_stream(const Kv8Call& c, const Kv8Parts& parts, cudaStream_t stream) {
  return c.dtype == APS_BF16 ? launch_typed<__nv_bfloat16>(c, parts, stream) : launch_typed<__half>(c, parts, stream);
}

}  // namespace aps
