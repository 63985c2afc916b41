// Up to 16 query rows per request over the 8-bit cache (kv8_common.cuh): decode, drafted tokens.  fp16 / bf16 queries, head sizes 64, 128.
//
// HBM-bound: the codes are read once, 2 D bytes a token and head.  One CTA of four warps per (request, head, part of the tokens); a warp
// takes every fourth group of 16 tokens (which never straddles a block), asynchronous copies bring its next groups to shared memory.
// The fragments of mma.sync.m16n8k16 are what plain vector loads of the rows give there, if the dimensions are counted in another order
// (a sum over them does not mind, and the output's columns are written where they belong):
//   S = Q K^T   B (16 dims x 8 tokens): lane (g, j) = (lane / 4, lane % 4) holds four codes of token g at a time, of its 16 consecutive
//               dims 16 j ... 16 j + 15 of a 64-byte half row; A holds the query's elements in the same order
//   O += P V    B (16 tokens x 8 dims): the lane holds tokens 2 j, 2 j + 1, 2 j + 8, 2 j + 9 of its D / 8 consecutive dims; a byte
//               permutation pairs the tokens, and tile i of the output has dim (D / 8) n + i in column n
// Every e4m3 number is an fp16 number.  The scales and the weights' two references are those of the tile kernel (kv8_prefix.cu).
#include "kv8_common.cuh"

#include <type_traits>

namespace aps {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kWarps = 4;
constexpr float kSlack = 8.f;   // log2 of how much the weights' reference may have grown before O is rescaled
constexpr float kUp = 7.f;      // log2 of what the weights are kept at

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 16 (or 4) bytes to shared memory; of which none: zeros.
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

template <int D> __host__ __device__ constexpr int stages() { return D == 128 ? 4 : 6; }   // groups of a warp in shared memory
template <int D> __host__ __device__ constexpr int stage_bytes() { return 2 * 16 * D + 16; }

// kHalves: of the 16 rows of a fragment, 1: up to 8 query rows, 2: up to 16.
template <typename T, int D, int kHalves>
__global__ void __launch_bounds__(kWarps * 32, kHalves == 1 ? 3 : 2)
kv8_stream_kernel(const Kv8Call c, const Kv8Parts parts, const uint32_t blocks_magic, const int vec) {
  constexpr int kCols = D / 64, kPer = D / 8, kStages = stages<D>();   // 64-byte pieces of a row; dims of a lane in V
  extern __shared__ __align__(128) uint8_t ring_raw[];                 // the warps' stages; in the end their outputs
  __shared__ float2 s_ml[kWarps][8 * kHalves];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
  const int head = blockIdx.x % c.cache.heads, part = blockIdx.x / c.cache.heads, req = part / parts.splits, split = part % parts.splits;
  if (blockIdx.x == 0 && threadIdx.x == 0) parts.plan[kPlanStatus] = kStatusOk;
  const int start = c.starts != nullptr ? c.starts[req] : req;
  const int rows_all = c.starts != nullptr ? c.starts[req + 1] - start : 1, n_rows = min(8 * kHalves, rows_all);
  if (n_rows <= 0) return;
  const int bs = c.cache.block_size, ctx = max(0, min(c.seq_lens[req], c.max_blocks * bs));
  const int first = ctx - rows_all;                    // own position of the first row
  const int all = (ctx + 15) / 16, per = (all + parts.splits - 1) / parts.splits;   // groups of 16 tokens
  const int group0 = min(all, split * per), n_groups = min(all, group0 + per) - group0;
  const int mine_groups = (n_groups - warp + kWarps - 1) / kWarps;                  // the warp's: warp, warp + 4, ...
  const int32_t* table = c.tables + (int64_t)req * c.max_blocks;
  const int64_t row_bytes = (int64_t)c.cache.heads * D;
  const uint32_t per_block = (uint32_t)bs / 16, ring = (uint32_t)__cvta_generic_to_shared(ring_raw) + warp * (kStages * stage_bytes<D>());
  auto block_at = [&](uint32_t group) { return blocks_magic ? __umulhi(group, blocks_magic) : group; };   // group / per_block
  auto block_of = [&](int k) { return k < mine_groups ? table[block_at(group0 + warp + k * kWarps)] : -1; };
  // the warp's group k on its way to stage k % kStages
  constexpr int kPieces = D / 16, kAtOnce = 32 / kPieces;
  auto fetch = [&](int k, int block) {
    const uint32_t group = group0 + warp + k * kWarps, to = ring + k % kStages * stage_bytes<D>();
    const bool in = block >= 0 && block < c.cache.num_blocks;
    if (!in) block = 0;   // something that can be read
    const int piece = lane % kPieces, r0 = lane / kPieces, live = in ? ctx - (int)group * 16 : 0;   // tokens that count
    const int64_t from = block * c.cache.block_stride + (int64_t)((group - block_at(group) * per_block) * 16 + r0) * row_bytes +
                         (int64_t)head * D + piece * 16;
#pragma unroll
    for (int i = 0; i < 16 / kAtOnce; ++i) copy16(to + piece_at<D>(r0 + i * kAtOnce, piece), c.cache.key + from + i * kAtOnce * row_bytes, r0 + i * kAtOnce < live);
#pragma unroll
    for (int i = 0; i < 16 / kAtOnce; ++i)
      copy16(to + 16 * D + piece_at<D>(r0 + i * kAtOnce, piece), c.cache.value + from + i * kAtOnce * row_bytes, r0 + i * kAtOnce < live);
    if (lane < 2) {
      const uint32_t at = to + 2 * 16 * D + 4 * lane;
      const int64_t place = block * c.cache.scale_stride + head;
      if (in) copy4(at, (lane == 0 ? c.cache.key_scale : c.cache.value_scale) + place);
      else asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(lane == 0 ? __int_as_float(0x7fc00000) : 0.f) : "memory");   // NaN scores
    }
  };
  int next = block_of(0);
#pragma unroll
  for (int k = 0; k < kStages - 1; ++k) {
    if (k < mine_groups) fetch(k, next);
    copy_commit();
    next = block_of(k + 1);
  }

  // the query's fragments, rows g and g + 8: a half row's 16 dims of the lane, four at a time; bf16 as fp16 times a power of two per row
  uint32_t qa[D / 16][2 * kHalves];
  float coef[kHalves];
#pragma unroll
  for (int r = 0; r < kHalves; ++r) {
    const int row = g + 8 * r;
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
    coef[r] = parts.scale_log2 * up;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      qa[s][r] = half2_bits(x[4 * s] * down, x[4 * s + 1] * down);
      qa[s][kHalves + r] = half2_bits(x[4 * s + 2] * down, x[4 * s + 3] * down);
    }
  }

  float acc[kPer][4];   // rows g, g, g + 8, g + 8
#pragma unroll
  for (int i = 0; i < kPer; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
  float m[kHalves], l[kHalves], ref[kHalves];
#pragma unroll
  for (int r = 0; r < kHalves; ++r) { m[r] = ref[r] = -INFINITY; l[r] = 0.f; }

  auto consume = [&](int k) {
    const int t0 = (group0 + warp + k * kWarps) * 16;
    const uint32_t at = ring + k % kStages * stage_bytes<D>();
    const float2 scales = shared_pair(at + 2 * 16 * D);
    float s[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
      for (int h = 0; h < kCols; ++h) {
        const uint4 k4 = shared16(at + piece_at<D>(8 * t + g, 4 * h + j));
        const uint32_t w[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t* a = qa[4 * h + e];
          mma16816(s[t], a[0], kHalves == 2 ? a[1] : 0u, a[kHalves], kHalves == 2 ? a[3] : 0u, e4m3x2_to_f16x2((uint16_t)w[e]),
                   e4m3x2_to_f16x2((uint16_t)(w[e] >> 16)));
        }
      }
    }
    const float lv = log2f(scales.y);
    uint32_t p[2][2];   // [tokens' half][rows' half]
    const bool edge = t0 + 15 > first;   // some row does not attend to all of the tokens
    bool any = false;
    float down[kHalves];
#pragma unroll
    for (int r = 0; r < kHalves; ++r) {
      float by = coef[r] * scales.x;
      if (edge) {
        // -infinity times a factor that is 0 or NaN would be NaN: such a factor goes into the scores
        const int seen = first + g + 8 * r - t0;   // the last token that the row attends to
        const bool plain = by > 0.f;
        const float fill = by == 0.f ? 0.f : __int_as_float(0x7fc00000);
        if (!plain) by = 1.f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& x = s[t][2 * r + e];
            x = 8 * t + 2 * j + e > seen ? -INFINITY : plain ? x : fill;
          }
      }
      float top = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
      top = fmaxf(top, __shfl_xor_sync(kFull, top, 1));
      top = fmaxf(top, __shfl_xor_sync(kFull, top, 2)) * by;   // NaN counts as none
      const float m_new = fmaxf(m[r], top), r_new = fmaxf(-INFINITY, top + lv);
      const bool move = r_new > ref[r] && !(r_new - ref[r] <= kSlack);
      any = any || move;
      down[r] = move && ref[r] != -INFINITY ? ex2(ref[r] - r_new) : 1.f;
      if (move) ref[r] = r_new;
      const float shift = m_new == -INFINITY ? 0.f : m_new, base = shift - (ref[r] == -INFINITY ? 0.f : ref[r]) + kUp + lv;
      const float off = base < -60.f ? -60.f : base, from = off - shift;
      float x[4], sum = 0.f;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          x[2 * t + e] = ex2(fmaf(s[t][2 * r + e], by, from));
          sum += x[2 * t + e];
        }
      l[r] = fmaf(sum, ex2(-off), m[r] == -INFINITY ? 0.f : l[r] * ex2(m[r] - shift));
      m[r] = m_new;
      p[0][r] = half2_bits(x[0], x[1]);
      p[1][r] = half2_bits(x[2], x[3]);
    }
    if (__any_sync(kFull, any)) {
#pragma unroll
      for (int n = 0; n < kPer; ++n)
#pragma unroll
        for (int r = 0; r < kHalves; ++r) { acc[n][2 * r] *= down[r]; acc[n][2 * r + 1] *= down[r]; }
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
    for (int w = 0; w < kPer / 4; ++w) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t b0 = __byte_perm(v[0][w], v[1][w], e ? 0x7362 : 0x5140), b1 = __byte_perm(v[2][w], v[3][w], e ? 0x7362 : 0x5140);
#pragma unroll
        for (int o = 0; o < 2; ++o)
          mma16816(acc[4 * w + 2 * e + o], p[0][0], kHalves == 2 ? p[0][1] : 0u, p[1][0], kHalves == 2 ? p[1][1] : 0u,
                   e4m3x2_to_f16x2((uint16_t)(b0 >> 16 * o)), e4m3x2_to_f16x2((uint16_t)(b1 >> 16 * o)));
      }
    }
  };
  for (int k = 0; k < mine_groups; ++k) {
    copy_wait<kStages - 2>();
    __syncwarp();   // every lane's copies of group k are there, every lane has read group k - 1
    if (k + kStages - 1 < mine_groups) fetch(k + kStages - 1, next);
    copy_commit();
    next = block_of(k + kStages);
    consume(k);
  }
  copy_wait<0>();
  __syncthreads();
  float (*s_o)[8 * kHalves][D] = reinterpret_cast<float (*)[8 * kHalves][D]>(ring_raw);

  // the warps' shares, relative to 2^m
#pragma unroll
  for (int r = 0; r < kHalves; ++r) {
    const int row = g + 8 * r;
    l[r] += __shfl_xor_sync(kFull, l[r], 1);
    l[r] += __shfl_xor_sync(kFull, l[r], 2);
    const float by = ref[r] == -INFINITY ? 0.f : ex2(ref[r] - kUp - (m[r] == -INFINITY ? 0.f : m[r]));
    if (row < n_rows) {
#pragma unroll
      for (int n = 0; n < kPer; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) s_o[warp][row][(2 * j + e) * kPer + n] = acc[n][2 * r + e] * by;
      if (j == 0) s_ml[warp][row] = make_float2(m[r], l[r]);
    }
  }
  __syncthreads();
  for (int at = threadIdx.x; at < n_rows * D; at += kWarps * 32) {
    const int row = at / D, d = at % D;
    const int64_t t = (int64_t)start + row;
    if (t < 0 || t >= c.rows) continue;
    float top = -INFINITY, sum = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_ml[w][row].x);
    const float shift = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float by = ex2(s_ml[w][row].x - shift);
      sum = fmaf(by, s_ml[w][row].y, sum);
      x = fmaf(by, s_o[w][row][d], x);
    }
    const int64_t unit = (t * c.cache.heads + head) * parts.splits + split;
    if (parts.splits == 1) {
      static_cast<T*>(c.out)[t * c.out_stride + (int64_t)head * D + d] = Elem<T>::from_float(first + row < 0 ? 0.f : x / sum);
    } else {
      parts.acc[unit * D + d] = x;
      if (d == 0) parts.ml[unit] = make_float2(top, sum);
    }
  }
}

template <typename T, int D, int kHalves>
int launch(const Kv8Call& c, const Kv8Parts& parts, cudaStream_t stream) {
  static bool done[64] = {false};
  auto kernel = kv8_stream_kernel<T, D, kHalves>;
  constexpr int smem = kWarps * stages<D>() * stage_bytes<D>();
  static_assert(smem >= (int)sizeof(float) * kWarps * 8 * kHalves * D, "the outputs fit into the stages");
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
  kernel<<<(unsigned)grid, kWarps * 32, smem, stream>>>(c, parts, kv8_blocks_magic(c.cache.block_size),
                                                        aligned_to(c.query, 16) && c.query_stride % 8 == 0);
  return launch_status("kv8_stream_kernel");
}

template <typename T>
int launch_typed(const Kv8Call& c, const Kv8Parts& parts, cudaStream_t stream) {
  const bool two = c.max_rows > 8;
  if (c.cache.head_size == 128) return two ? launch<T, 128, 2>(c, parts, stream) : launch<T, 128, 1>(c, parts, stream);
  return two ? launch<T, 64, 2>(c, parts, stream) : launch<T, 64, 1>(c, parts, stream);
}

}  // namespace

bool kv8_stream_takes(const Kv8Call& c) {
  return (c.starts == nullptr || c.max_rows <= 16) && (c.dtype == APS_F16 || c.dtype == APS_BF16) &&
         (c.cache.head_size == 64 || c.cache.head_size == 128) && c.cache.num_blocks > 0 && c.scale >= 1.17549435e-38f && c.scale < 1.70141183e38f;
}

// Parts that a request's tokens are cut into: enough CTAs for eight per SM, 256 tokens of the tables' width each at least.
int kv8_stream_splits(const Kv8Call& c) {
  const int64_t units = (int64_t)c.batch * c.cache.heads, tokens = (int64_t)c.max_blocks * c.cache.block_size;
  const int64_t want = ((int64_t)sm_count() * 8 + units - 1) / units, most = (tokens + 255) / 256;
  const int64_t n = want < most ? want : most;
  return (int)(n < 1 ? 1 : n > 1024 ? 1024 : n);
}

int launch_kv8_stream(const Kv8Call& c, const Kv8Parts& parts, cudaStream_t stream) {
  return c.dtype == APS_BF16 ? launch_typed<__nv_bfloat16>(c, parts, stream) : launch_typed<__half>(c, parts, stream);
}

}  // namespace aps
