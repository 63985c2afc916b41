// Up to 16 query rows per request over the 8-bit cache (kv8_common.cuh): decode, drafted tokens.  fp16 / bf16 queries, head sizes 64, 128.
//
// HBM-bound: the codes are read once, 2 D bytes a token and head.  One CTA of four warps per (request, head, part of the tokens); a warp
// takes every fourth group of 16 tokens (which never straddles a block), its next groups already on their way to registers.  No shared
// memory in between: the fragments of mma.sync.m16n8k16 are what 16-byte loads of the cache's rows give, if the dimensions are counted
// in another order (a sum over them does not mind, and the output's columns are written where they belong):
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
// Loads that stay ahead of what is computed between them and their use.
__device__ __forceinline__ void ld_ahead(const uint8_t* p, uint4& v) {
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
}
__device__ __forceinline__ void ld_ahead(const uint8_t* p, uint2& v) {
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
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

// kHalves: of the 16 rows of a fragment, 1: up to 8 query rows, 2: up to 16.
template <typename T, int D, int kHalves>
__global__ void __launch_bounds__(kWarps * 32, kHalves == 1 ? 3 : 2)
kv8_stream_kernel(const Kv8Call c, const Kv8Parts parts, const uint32_t blocks_magic, const int vec) {
  constexpr int kCols = D / 64, kPer = D / 8;          // 64-byte pieces of a row; dims of a lane in V
  constexpr int kAhead = D == 128 ? 2 : 4;             // groups of a warp in flight
  using V = typename std::conditional<D == 128, uint4, uint2>::type;
  struct Group { uint4 k[2][kCols]; V v[4]; float key_scale, value_scale; };
  __shared__ float s_o[kWarps][8 * kHalves][D];
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
  const int32_t* table = c.tables + (int64_t)req * c.max_blocks;
  const int64_t row_bytes = (int64_t)c.cache.heads * D;
  const uint32_t per_block = (uint32_t)bs / 16;
  auto block_at = [&](uint32_t group) { return blocks_magic ? __umulhi(group, blocks_magic) : group; };   // group / per_block
  auto block_of = [&](int i) { return i < n_groups ? table[block_at(group0 + i)] : -1; };
  auto load = [&](Group& f, int i, int block) {
    const uint32_t group = group0 + i;
    const bool in = block >= 0 && block < c.cache.num_blocks;
    if (!in) block = 0;   // something that can be read
    const int64_t from = block * c.cache.block_stride + (int64_t)((group - block_at(group) * per_block) * 16) * row_bytes + (int64_t)head * D;
    const uint8_t *k = c.cache.key + from + g * row_bytes + j * 16, *v = c.cache.value + from + 2 * j * row_bytes + g * kPer;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int h = 0; h < kCols; ++h) ld_ahead(k + 8 * t * row_bytes + 64 * h, f.k[t][h]);
#pragma unroll
    for (int t = 0; t < 4; ++t) ld_ahead(v + ((t & 1) + 8 * (t >> 1)) * row_bytes, f.v[t]);
    const int64_t at = block * c.cache.scale_stride + head;
    // a block outside the cache: the scores of its tokens are NaN
    f.key_scale = in ? c.cache.key_scale[at] : __int_as_float(0x7fc00000);
    f.value_scale = in ? c.cache.value_scale[at] : 0.f;
  };
  Group buf[kAhead];
  int next = block_of(warp);
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    if (warp + u * kWarps < n_groups) load(buf[u], warp + u * kWarps, next);
    next = block_of(warp + (u + 1) * kWarps);
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

  auto consume = [&](Group& f, int i) {
    const int t0 = (group0 + i) * 16;
    float s[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
      for (int h = 0; h < kCols; ++h) {
        const uint32_t w[4] = {f.k[t][h].x, f.k[t][h].y, f.k[t][h].z, f.k[t][h].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t* a = qa[4 * h + e];
          mma16816(s[t], a[0], kHalves == 2 ? a[1] : 0u, a[kHalves], kHalves == 2 ? a[3] : 0u, e4m3x2_to_f16x2((uint16_t)w[e]),
                   e4m3x2_to_f16x2((uint16_t)(w[e] >> 16)));
        }
      }
    }
    const float lv = log2f(f.value_scale);
    uint32_t p[2][2];   // [tokens' half][rows' half]
    const bool edge = t0 + 15 > first;   // some row does not attend to all of the tokens
    bool any = false;
    float down[kHalves];
#pragma unroll
    for (int r = 0; r < kHalves; ++r) {
      float by = coef[r] * f.key_scale;
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
    if (t0 + 16 > ctx) {   // rows behind the last token have no weight, but zero times whatever they hold might be NaN
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (t0 + 2 * j + (t & 1) + 8 * (t >> 1) >= ctx) f.v[t] = V{};
    }
    const uint32_t* v[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) v[t] = reinterpret_cast<const uint32_t*>(&f.v[t]);
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
  for (int i = warp; i < n_groups; i += kAhead * kWarps) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int at = i + u * kWarps;
      if (at < n_groups) {
        consume(buf[u], at);
        if (at + kAhead * kWarps < n_groups) load(buf[u], at + kAhead * kWarps, next);
        next = block_of(at + (kAhead + 1) * kWarps);
      }
    }
  }

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
  const int64_t grid = (int64_t)c.batch * parts.splits * c.cache.heads;
  APS_REQUIRE(grid < (int64_t(1) << 31), APS_ERR_SHAPE, "kv8_attention: too many requests");
  kv8_stream_kernel<T, D, kHalves><<<(unsigned)grid, kWarps * 32, 0, stream>>>(c, parts, kv8_blocks_magic(c.cache.block_size),
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
