// Attention over the 8-bit cache (kv8_common.cuh), any number of query rows per request.
//
//   kv8_rows_kernel     CUDA-core arithmetic, one CTA per (query row, head, part of the row's tokens): every query type, head size
//                       and block stride.  D / 16 lanes cover a row with one 16-byte load each.
//   (kv8_stream.cu)     up to 16 query rows per request, HBM-bound
//   (kv8_prefix.cu)     several query rows per request on the tensor cores
//   kv8_combine_kernel  joins the parts of rows whose tokens were cut.
// Scores, softmax statistics and sums are fp32; a code times its scale is exact in fp32.
#include "kv8_common.cuh"

#include <initializer_list>

namespace aps {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kRowWarps = 4;

template <typename T, int D>
__global__ void __launch_bounds__(kRowWarps * 32)
kv8_rows_kernel(const Kv8Call c, const Kv8Parts a) {
  constexpr int kLanes = D / 16, kTok = 32 / kLanes, kLoads = 4;   // lanes per row, rows per load, loads at a time
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane % kLanes, tsel = lane / kLanes;
  chain_wait();
  chain_next();
  const int64_t t = blockIdx.x / a.splits;
  const int split = (int)(blockIdx.x % a.splits), h = blockIdx.y;
  if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) a.plan[kPlanStatus] = kStatusOk;
  int req, keys;
  if (!kv8_find_row(c, t, req, keys)) return;
  const int per = ((keys + a.splits - 1) / a.splits + 15) / 16 * 16;
  const int begin = min(keys, split * per), end = min(keys, begin + per);
  const int32_t* table = c.tables + (int64_t)req * c.max_blocks;
  const int64_t row_bytes = (int64_t)c.cache.heads * D;

  float q[16];
  {
    const T* src = static_cast<const T*>(c.query) + t * c.query_stride + (int64_t)h * D + sub * 16;
#pragma unroll
    for (int i = 0; i < 16; ++i) q[i] = Elem<T>::to_float(src[i]) * a.scale_log2;
  }
  float acc[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
  float m = -INFINITY, l = 0.f;
  for (int t0 = begin + warp * kTok * kLoads; t0 < end; t0 += kRowWarps * kTok * kLoads) {
    uint4 kr[kLoads], vr[kLoads];
    float ks[kLoads], vs[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int tok = t0 + i * kTok + tsel;
      kr[i] = vr[i] = make_uint4(0, 0, 0, 0);
      ks[i] = vs[i] = __int_as_float(0x7fc00000);   // a block outside the cache: the row becomes NaN
      if (tok < end) {
        const int64_t block = table[tok / c.cache.block_size];
        if (block >= 0 && block < c.cache.num_blocks) {
          const int64_t at = block * c.cache.block_stride + tok % c.cache.block_size * row_bytes + (int64_t)h * D + sub * 16;
          kr[i] = *reinterpret_cast<const uint4*>(c.cache.key + at);
          vr[i] = *reinterpret_cast<const uint4*>(c.cache.value + at);
          ks[i] = c.cache.key_scale[block * c.cache.scale_stride + h];
          vs[i] = c.cache.value_scale[block * c.cache.scale_stride + h];
        }
      } else {
        vs[i] = 0.f;
      }
    }
    float s[kLoads], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      float k[16], x = 0.f;
      e4m3x4_to_float(kr[i].x, k); e4m3x4_to_float(kr[i].y, k + 4); e4m3x4_to_float(kr[i].z, k + 8); e4m3x4_to_float(kr[i].w, k + 12);
#pragma unroll
      for (int e = 0; e < 16; ++e) x = fmaf(q[e], k[e], x);
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) x += __shfl_xor_sync(kFull, x, o);
      s[i] = t0 + i * kTok + tsel < end ? x * ks[i] : -INFINITY;
      top = fmaxf(top, s[i]);
    }
#pragma unroll
    for (int o = kLanes; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
    const float now = fmaxf(m, top), ref = now == -INFINITY ? 0.f : now, down = exp2f(m - ref);
    l *= down;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] *= down;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const float p = exp2f(s[i] - ref), w = p * vs[i];
      l += p;
      float v[16];
      e4m3x4_to_float(vr[i].x, v); e4m3x4_to_float(vr[i].y, v + 4); e4m3x4_to_float(vr[i].z, v + 8); e4m3x4_to_float(vr[i].w, v + 12);
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[e] = fmaf(w, v[e], acc[e]);
    }
    m = now;
  }
#pragma unroll
  for (int o = kLanes; o < 32; o <<= 1) {
    l += __shfl_xor_sync(kFull, l, o);
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] += __shfl_xor_sync(kFull, acc[e], o);
  }
  // the warps' shares, in order
  __shared__ float s_acc[kRowWarps][D];
  __shared__ float2 s_ml[kRowWarps];
  if (tsel == 0) {
#pragma unroll
    for (int e = 0; e < 16; ++e) s_acc[warp][sub * 16 + e] = acc[e];
    if (lane == 0) s_ml[warp] = make_float2(m, l);
  }
  __syncthreads();
  float top = -INFINITY, sum = 0.f, w[kRowWarps];
#pragma unroll
  for (int i = 0; i < kRowWarps; ++i) top = fmaxf(top, s_ml[i].x);
  const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int i = 0; i < kRowWarps; ++i) { w[i] = exp2f(s_ml[i].x - ref); sum = fmaf(w[i], s_ml[i].y, sum); }
  const int64_t unit = (t * c.cache.heads + h) * a.splits + split;
  for (int d = threadIdx.x; d < D; d += kRowWarps * 32) {
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < kRowWarps; ++i) x = fmaf(w[i], s_acc[i][d], x);
    if (a.splits == 1)
      static_cast<T*>(c.out)[t * c.out_stride + (int64_t)h * D + d] = Elem<T>::from_float(keys == 0 ? 0.f : x / sum);
    else
      a.acc[unit * D + d] = x;
  }
  if (a.splits > 1 && threadIdx.x == 0) a.ml[unit] = make_float2(top, sum);
}

// One CTA per (query row, head): the parts' weights first, then D / 4 lanes take four elements of the output each, the others share the
// parts.  Always in the same order.  (A warp per row took 18 us over 118 parts of one row, one part after the other.)
constexpr int kMostParts = 1024;

template <typename T, int D>
__global__ void __launch_bounds__(128)
kv8_combine_kernel(const Kv8Call c, const Kv8Parts a) {
  constexpr int kLanes = D / 4, kShare = 128 / kLanes;
  __shared__ float s_w[kMostParts];
  __shared__ float s_red[2][4];
  __shared__ __align__(16) float4 s_x[128];
  chain_wait();
  chain_next();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, d = tid % kLanes * 4, share = tid / kLanes;
  const int64_t unit = blockIdx.x, t = unit / c.cache.heads, h = unit % c.cache.heads;
  int req, keys;
  if (!kv8_find_row(c, t, req, keys)) return;
  const float2* ml = a.ml + unit * a.splits;
  const float* acc = a.acc + unit * a.splits * D + d;
  float top = -INFINITY, sum = 0.f;
  for (int i = tid; i < a.splits; i += 128) top = fmaxf(top, ml[i].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
  if (lane == 0) s_red[0][warp] = top;
  __syncthreads();
  top = fmaxf(fmaxf(s_red[0][0], s_red[0][1]), fmaxf(s_red[0][2], s_red[0][3]));
  const float ref = top == -INFINITY ? 0.f : top;
  for (int i = tid; i < a.splits; i += 128) {
    const float2 x = ml[i];
    const float w = exp2f(x.x - ref);
    sum = fmaf(w, x.y, sum);
    s_w[i] = x.x == -INFINITY ? -1.f : w;   // no acc: no tokens, or scores that are all NaN (0 times its sum is NaN then, too)
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
  if (lane == 0) s_red[1][warp] = sum;
  __syncthreads();
  sum = (s_red[1][0] + s_red[1][1]) + (s_red[1][2] + s_red[1][3]);
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = share; i < a.splits; i += kShare) {
    const float w = s_w[i];
    const float4 y = w < 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : *reinterpret_cast<const float4*>(acc + (int64_t)i * D);
    x.x = fmaf(w, y.x, x.x); x.y = fmaf(w, y.y, x.y); x.z = fmaf(w, y.z, x.z); x.w = fmaf(w, y.w, x.w);
  }
  s_x[tid] = x;
  __syncthreads();
  if (share == 0) {
#pragma unroll
    for (int i = 1; i < kShare; ++i) {
      const float4 y = s_x[tid + i * kLanes];
      x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
    }
    const float y[4] = {x.x, x.y, x.z, x.w};
    T* out = static_cast<T*>(c.out) + t * c.out_stride + h * D + d;
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = Elem<T>::from_float(keys == 0 ? 0.f : y[e] / sum);
  }
}

// A few parts: one warp per (query row, head), all loads at once (256 OPT-13B requests of four parts: 15 us with the kernel above, 8 with this one).
constexpr int kFewParts = 8;

template <typename T, int D>
__global__ void __launch_bounds__(256)
kv8_combine_few_kernel(const Kv8Call c, const Kv8Parts a) {
  constexpr int kPer = D / 32;
  chain_wait();
  chain_next();
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (unit >= c.rows * c.cache.heads) return;
  const int64_t t = unit / c.cache.heads, h = unit % c.cache.heads;
  struct alignas(kPer * 4 > 16 ? 16 : kPer * 4) Piece { float x[kPer]; };
  float2 ml[kFewParts];
  Piece y[kFewParts];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kFewParts; ++i) {
    ml[i] = i < a.splits ? a.ml[unit * a.splits + i] : make_float2(-INFINITY, 0.f);
    if (i < a.splits) y[i] = *reinterpret_cast<const Piece*>(a.acc + (unit * a.splits + i) * D + lane * kPer);
    top = fmaxf(top, ml[i].x);
  }
  int req, keys;
  if (!kv8_find_row(c, t, req, keys)) return;
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f, x[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) x[e] = 0.f;
#pragma unroll
  for (int i = 0; i < kFewParts; ++i) {
    if (ml[i].x == -INFINITY) {   // no acc: a part without tokens, whose sum is 0, or one whose scores are all NaN, whose sum is NaN
      sum += ml[i].y;
      continue;
    }
    const float w = exp2f(ml[i].x - ref);
    sum = fmaf(w, ml[i].y, sum);
#pragma unroll
    for (int e = 0; e < kPer; ++e) x[e] = fmaf(w, y[i].x[e], x[e]);
  }
  T* out = static_cast<T*>(c.out) + t * c.out_stride + h * D + lane * kPer;
#pragma unroll
  for (int e = 0; e < kPer; ++e) out[e] = Elem<T>::from_float(keys == 0 ? 0.f : x[e] / sum);
}

// Parts a row's tokens are cut into: enough CTAs for the GPU, parts of 512 tokens at least (joining them takes a launch).
int row_splits(const Kv8Call& c) {
  const int64_t units = c.rows * c.cache.heads, tokens = (int64_t)c.max_blocks * c.cache.block_size;
  const int64_t want = ((int64_t)sm_count() * 8 + units - 1) / units, most = (tokens + 511) / 512;
  const int64_t n = want < most ? want : most;
  return (int)(n < 1 ? 1 : n > kMostParts ? kMostParts : n);
}

// The scratch: header, maxima and sums, weighted values (16-byte stores).
size_t part_acc_at(int64_t rows, int heads, int splits) {
  return align_up(kPlanWords * sizeof(int) + (size_t)rows * heads * splits * sizeof(float2), 256);
}
size_t part_scratch(int64_t rows, int heads, int head_size, int splits) {
  if (splits == 1) return kPlanWords * sizeof(int);
  return part_acc_at(rows, heads, splits) + (size_t)rows * heads * splits * head_size * sizeof(float);
}

template <typename T>
int launch_parts_combine(const Kv8Call& c, const Kv8Parts& a, cudaStream_t stream) {
  if (a.splits == 1) return APS_OK;
  const int64_t grid = c.rows * c.cache.heads;
  APS_REQUIRE(grid < (int64_t(1) << 31), APS_ERR_SHAPE, "kv8_attention: too many rows");
  if (a.splits <= kFewParts) {
    const unsigned few = (unsigned)((grid + 7) / 8);
    switch (c.cache.head_size) {
      case 32: return launch_chained("kv8_combine_few_kernel", kv8_combine_few_kernel<T, 32>, few, 256, 0, stream, c, a);
      case 64: return launch_chained("kv8_combine_few_kernel", kv8_combine_few_kernel<T, 64>, few, 256, 0, stream, c, a);
      case 128: return launch_chained("kv8_combine_few_kernel", kv8_combine_few_kernel<T, 128>, few, 256, 0, stream, c, a);
      default: return launch_chained("kv8_combine_few_kernel", kv8_combine_few_kernel<T, 256>, few, 256, 0, stream, c, a);
    }
  }
  switch (c.cache.head_size) {
    case 32: return launch_chained("kv8_combine_kernel", kv8_combine_kernel<T, 32>, (unsigned)grid, 128, 0, stream, c, a);
    case 64: return launch_chained("kv8_combine_kernel", kv8_combine_kernel<T, 64>, (unsigned)grid, 128, 0, stream, c, a);
    case 128: return launch_chained("kv8_combine_kernel", kv8_combine_kernel<T, 128>, (unsigned)grid, 128, 0, stream, c, a);
    default: return launch_chained("kv8_combine_kernel", kv8_combine_kernel<T, 256>, (unsigned)grid, 128, 0, stream, c, a);
  }
}

template <typename T, int D>
int launch_rows(const Kv8Call& c, const Kv8Parts& a, cudaStream_t stream) {
  const int64_t grid = c.rows * a.splits;
  APS_REQUIRE(grid < (int64_t(1) << 31), APS_ERR_SHAPE, "kv8_attention: too many rows");
  return launch_chained("kv8_rows_kernel", kv8_rows_kernel<T, D>, dim3((unsigned)grid, c.cache.heads), kRowWarps * 32, 0, stream, c, a);
}

enum Way { kRows, kStream, kTiles };

Way way_of(const Kv8Call& c) { return kv8_stream_takes(c) ? kStream : kv8_tiles_take(c) ? kTiles : kRows; }
int splits_of(const Kv8Call& c, Way way) { return way == kStream ? kv8_stream_splits(c) : way == kTiles ? kv8_tile_splits(c) : row_splits(c); }

template <typename T>
int attend(const Kv8Call& c, const Kv8Parts& a, Way way, cudaStream_t stream) {
  int st;
  if (way == kStream) {
    st = launch_kv8_stream(c, a, stream);
  } else if (way == kTiles) {
    st = launch_kv8_tiles(c, a, stream);
  } else {
    switch (c.cache.head_size) {
      case 32: st = launch_rows<T, 32>(c, a, stream); break;
      case 64: st = launch_rows<T, 64>(c, a, stream); break;
      case 128: st = launch_rows<T, 128>(c, a, stream); break;
      default: st = launch_rows<T, 256>(c, a, stream); break;
    }
  }
  return st != APS_OK ? st : launch_parts_combine<T>(c, a, stream);
}

int check_call(const char* op, const Kv8Call& c) {
  const int st = check_kv8_cache(op, c.cache, c.dtype);
  if (st != APS_OK) return st;
  APS_REQUIRE(c.batch >= 0 && c.rows >= 0 && c.max_blocks > 0 && c.max_rows >= 0, APS_ERR_SHAPE, "%s: bad sizes", op);
  APS_REQUIRE((int64_t)c.max_blocks * c.cache.block_size < (int64_t(1) << 30) && c.rows < (int64_t(1) << 31), APS_ERR_SHAPE,
              "%s: tables for more than 2^30 tokens", op);
  if (c.rows == 0 || c.batch == 0) return APS_OK;
  APS_REQUIRE(c.out && c.query && c.tables && c.seq_lens && c.cache.key && c.cache.value && c.cache.key_scale && c.cache.value_scale,
              APS_ERR_NULL_POINTER, "%s: null pointer", op);
  const int es = dtype_size(c.dtype);
  const int64_t row = (int64_t)c.cache.heads * c.cache.head_size;
  APS_REQUIRE(c.query_stride >= row && c.out_stride >= row, APS_ERR_SHAPE, "%s: strides smaller than a row", op);
  APS_REQUIRE(aligned_to(c.query, es) && aligned_to(c.out, es) && aligned_to(c.cache.key, 16) && aligned_to(c.cache.value, 16) &&
                  c.cache.block_stride % 16 == 0 && aligned_to(c.cache.key_scale, 4) && aligned_to(c.cache.value_scale, 4) &&
                  aligned_to(c.tables, 4) && aligned_to(c.seq_lens, 4) && aligned_to(c.starts, 4),
              APS_ERR_MISALIGNED, "%s: the caches must be 16-byte aligned with blocks at multiples of 16 bytes", op);
  return APS_OK;
}

}  // namespace
}  // namespace aps

using namespace aps;

extern "C" size_t aps_kv8_attention_workspace_bytes(int batch, int64_t num_rows, int max_query_len, int max_blocks_per_seq, int block_size,
                                                    int num_heads, int head_size, int dtype) {
  if (batch <= 0 || num_rows <= 0 || max_query_len < 0 || max_blocks_per_seq <= 0 || block_size <= 0 || num_heads <= 0 || head_size <= 0) return 0;
  Kv8Call c{};
  c.batch = batch; c.rows = num_rows; c.max_rows = max_query_len < num_rows ? max_query_len : (int)num_rows; c.max_blocks = max_blocks_per_seq;
  c.cache.heads = num_heads; c.cache.head_size = head_size; c.cache.block_size = block_size; c.cache.num_blocks = 1;
  c.scale = 1.f; c.dtype = dtype;
  // what the kernel takes that such a call runs: with a scale that is not positive the CUDA-core one, with starts or (a row for each
  // request) without
  const int32_t some = 0;
  int most = row_splits(c);
  for (const int32_t* starts : {(const int32_t*)nullptr, &some}) {
    if (starts == nullptr && num_rows != batch) continue;
    c.starts = starts;
    const int splits = splits_of(c, way_of(c));
    most = splits > most ? splits : most;
  }
  return part_scratch(num_rows, num_heads, head_size, most);
}

namespace aps {
namespace {

// The call as it will run, or what is wrong with it.
int plan_attention(const Kv8Call& c, void* workspace, size_t workspace_bytes, Way* way, Kv8Parts* a) {
  const int st = check_call("kv8_attention", c);
  if (st != APS_OK || c.rows == 0 || c.batch == 0) return st;
  APS_REQUIRE(c.starts != nullptr || c.rows == c.batch, APS_ERR_SHAPE, "kv8_attention: %lld query rows for %d requests",
              (long long)c.rows, c.batch);
  *way = way_of(c);
  const int splits = splits_of(c, *way);
  *a = Kv8Parts{static_cast<int*>(workspace), nullptr, nullptr, splits, c.scale * 1.4426950408889634f};
  const size_t need = part_scratch(c.rows, c.cache.heads, c.cache.head_size, splits);
  APS_REQUIRE(workspace != nullptr && aligned_to(workspace, 256) && workspace_bytes >= need, APS_ERR_WORKSPACE,
              "kv8_attention: workspace must be 256-byte aligned and hold %zu bytes (got %zu)", need, workspace_bytes);
  if (splits > 1) {
    a->ml = reinterpret_cast<float2*>(a->plan + kPlanWords);
    a->acc = reinterpret_cast<float*>(static_cast<char*>(workspace) + part_acc_at(c.rows, c.cache.heads, splits));
  }
  return APS_OK;
}

int run_attention(const Kv8Call& c, Way way, const Kv8Parts& a, cudaStream_t stream) {
  if (c.rows == 0 || c.batch == 0) return APS_OK;
  switch (c.dtype) {
    case APS_F32: return attend<float>(c, a, way, stream);
    case APS_F16: return attend<__half>(c, a, way, stream);
    default: return attend<__nv_bfloat16>(c, a, way, stream);
  }
}

}  // namespace
}  // namespace aps

extern "C" int aps_kv8_attention(void* out, const void* query, const void* key_cache, const void* value_cache, const float* key_scale,
                                 const float* value_scale, const int32_t* block_tables, const int32_t* query_start_loc,
                                 const int32_t* seq_lens, int batch, int64_t num_rows, int max_query_len, int max_blocks_per_seq,
                                 int num_heads, int head_size, int block_size, int64_t num_blocks, int64_t query_stride,
                                 int64_t out_stride, int64_t block_stride, int64_t scale_stride, float scale, void* workspace,
                                 size_t workspace_bytes, int dtype, void* stream) {
  const Kv8Call c{out, query,
                  {(const uint8_t*)key_cache, (const uint8_t*)value_cache, key_scale, value_scale, num_blocks, block_stride, scale_stride,
                   num_heads, head_size, block_size},
                  block_tables, query_start_loc, seq_lens, batch, max_blocks_per_seq,
                  max_query_len < num_rows ? max_query_len : (int)num_rows, num_rows, query_stride, out_stride, scale, dtype};
  Way way = kRows;
  Kv8Parts a{};
  const int st = plan_attention(c, workspace, workspace_bytes, &way, &a);
  return st != APS_OK ? st : run_attention(c, way, a, (cudaStream_t)stream);
}

extern "C" int aps_kv8_decode_step(void* out, const void* query, const void* key, const void* value, void* key_cache, void* value_cache,
                                   float* key_scale, float* value_scale, const int64_t* slot_mapping, int64_t num_slots,
                                   const int32_t* block_tables, const int32_t* seq_lens, int batch, int max_blocks_per_seq, int num_heads,
                                   int head_size, int block_size, int64_t num_blocks, int64_t query_stride, int64_t key_stride,
                                   int64_t value_stride, int64_t out_stride, int64_t block_stride, int64_t scale_stride, float scale,
                                   void* workspace, size_t workspace_bytes, int dtype, void* stream) {
  const Kv8Call c{out, query,
                  {(const uint8_t*)key_cache, (const uint8_t*)value_cache, key_scale, value_scale, num_blocks, block_stride, scale_stride,
                   num_heads, head_size, block_size},
                  block_tables, nullptr, seq_lens, batch, max_blocks_per_seq, 1, batch, query_stride, out_stride, scale, dtype};
  Way way = kRows;
  Kv8Parts a{};
  int st = plan_attention(c, workspace, workspace_bytes, &way, &a);   // before anything is written
  if (st != APS_OK) return st;
  st = aps_kv8_write(key, value, key_cache, value_cache, key_scale, value_scale, slot_mapping, num_slots, num_heads, head_size, block_size,
                     num_blocks, key_stride, value_stride, block_stride, scale_stride, workspace, workspace_bytes, dtype, stream);
  return st != APS_OK ? st : run_attention(c, way, a, (cudaStream_t)stream);
}
