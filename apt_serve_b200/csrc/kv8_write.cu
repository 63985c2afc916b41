// Rows of K and V into the 8-bit cache (kv8_common.cuh).
//
// Stands beside aps_reshape_and_cache, with the same slots: slot / BS is the block, slot % BS the row in it.  All rows of a call that
// go to one block are taken together, whatever their order in the mapping (of two rows for one slot the later one stays).  If the
// block's first slot is among them the block starts anew: its scale is that of the new rows, its other rows are left as they are.
// Otherwise the block's scale becomes the larger of the old one and the new rows', and, where it grows, the block's other rows are
// rounded to it.
//
// What bounds it: bytes, (element size + 1) for each element of prompts' rows; launch and two round trips for single tokens.
#include "kv8_common.cuh"

namespace aps {
namespace {

constexpr int kThreads = 256;

__device__ int g_kv8_status = 0;   // a slot past the cache has been met since this was read last

struct WriteArgs {
  const void* rows[2];        // key, value
  uint8_t* cache[2];
  float* scale[2];
  const int64_t* slots;
  int64_t tokens, num_blocks, row_stride[2], block_stride, scale_stride;
  int heads, block_size;
};

template <int D> struct RowCfg {
  static constexpr int kPer = D == 256 ? 8 : 4;     // elements per lane
  static constexpr int kLanes = D / kPer;           // lanes per row
  static constexpr int kRows = 32 / kLanes;         // rows a warp has at a time
};

// kPer elements as floats.
template <typename T, int N, bool kAligned>
__device__ __forceinline__ void load_elements(const T* p, float* f) {
  if constexpr (kAligned) {
    struct alignas(N * sizeof(T) > 16 ? 16 : N * sizeof(T)) Pack { T x[N]; };
    const Pack v = *reinterpret_cast<const Pack*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = Elem<T>::to_float(v.x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = Elem<T>::to_float(p[i]);
  }
}

// One head of one plane of a block, by one warp: token[o] is the row that goes to slot o of the block, -1 for none.
template <typename T, int D, bool kAligned>
__device__ __forceinline__ void write_head(const WriteArgs& a, int plane, int head, int64_t block, const int* token, int lane) {
  using C = RowCfg<D>;
  const T* rows = static_cast<const T*>(a.rows[plane]) + (int64_t)head * D + lane % C::kLanes * C::kPer;
  uint8_t* held = a.cache[plane] + block * a.block_stride + (int64_t)head * D + lane % C::kLanes * C::kPer;
  const int64_t held_row = (int64_t)a.heads * D;
  float* scale_at = a.scale[plane] + block * a.scale_stride + head;
  const float old = *scale_at;
  const bool anew = token[0] >= 0;
  float top = 0.f;
  for (int o = lane / C::kLanes; o < a.block_size; o += C::kRows) {
    if (token[o] < 0) continue;
    float x[C::kPer];
    load_elements<T, C::kPer, kAligned>(rows + token[o] * a.row_stride[plane], x);
#pragma unroll
    for (int i = 0; i < C::kPer; ++i)
      if (fabsf(x[i]) <= 3.402823466e38f) top = fmaxf(top, fabsf(x[i]));   // not NaN, not infinite
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float need = e4m3_scale(top), s = anew ? need : fmaxf(old, need);
  const bool shift = (__float_as_uint(s) & 0x7fffffu) == 0;   // a power of two: its reciprocal is exact
  const float inv = 1.f / s, ratio = old / s;
  const bool move = !anew && s != old;
  for (int o = lane / C::kLanes; o < a.block_size; o += C::kRows) {
    uint32_t* to = reinterpret_cast<uint32_t*>(held + o * held_row);
    if (token[o] >= 0) {
      float x[C::kPer];
      load_elements<T, C::kPer, kAligned>(rows + token[o] * a.row_stride[plane], x);
#pragma unroll
      for (int i = 0; i < C::kPer; ++i) {
        const float y = shift ? x[i] * inv : x[i] / s;
        x[i] = fabsf(x[i]) <= 3.402823466e38f ? y : __int_as_float(0x7fc00000);
      }
#pragma unroll
      for (int i = 0; i < C::kPer / 4; ++i) to[i] = float4_to_e4m3x4(x + 4 * i);
    } else if (move) {
#pragma unroll
      for (int i = 0; i < C::kPer / 4; ++i) {
        float x[4];
        e4m3x4_to_float(to[i], x);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] *= ratio;
        to[i] = float4_to_e4m3x4(x);
      }
    }
  }
  if (lane == 0 && s != old) *scale_at = s;
}

// One CTA per (row, some heads); the CTA of the first row of a block does the block.
template <typename T, int D, bool kAligned>
__global__ void __launch_bounds__(kThreads)
kv8_write_kernel(const WriteArgs a) {
  extern __shared__ int token[];   // [block_size]
  __shared__ int s_later;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t t = blockIdx.x, slot = a.slots[t];
  if (slot < 0) return;
  const int64_t block = slot / a.block_size;
  if (block >= a.num_blocks) {
    if (tid == 0) g_kv8_status = kStatusBadIndex;
    return;
  }
  auto same = [&](int64_t other) { return other >= 0 && other / a.block_size == block; };
  if (t > 0 && same(a.slots[t - 1])) return;
  for (int o = tid; o < a.block_size; o += kThreads) token[o] = -1;
  if (tid == 0) s_later = 0;
  __syncthreads();
  for (int64_t i = tid; i < a.tokens; i += kThreads) {
    const int64_t other = a.slots[i];
    if (!same(other)) continue;
    if (i < t) s_later = 1;
    atomicMax(&token[other % a.block_size], (int)i);
  }
  __syncthreads();
  if (s_later) return;
  for (int u = blockIdx.y * (kThreads / 32) + warp; u < 2 * a.heads; u += gridDim.y * (kThreads / 32))
    write_head<T, D, kAligned>(a, u >= a.heads, u >= a.heads ? u - a.heads : u, block, token, lane);
}

template <typename T, int D>
int launch_write(const WriteArgs& a, bool aligned, cudaStream_t stream) {
  auto kernel = aligned ? kv8_write_kernel<T, D, true> : kv8_write_kernel<T, D, false>;
  const dim3 grid((unsigned)a.tokens, (2 * a.heads + kThreads / 32 - 1) / (kThreads / 32));
  kernel<<<grid, kThreads, a.block_size * sizeof(int), stream>>>(a);
  return launch_status("kv8_write_kernel");
}

template <typename T>
int write_by_head(const WriteArgs& a, int head_size, bool aligned, cudaStream_t stream) {
  switch (head_size) {
    case 32: return launch_write<T, 32>(a, aligned, stream);
    case 64: return launch_write<T, 64>(a, aligned, stream);
    case 128: return launch_write<T, 128>(a, aligned, stream);
    default: return launch_write<T, 256>(a, aligned, stream);
  }
}

}  // namespace

int read_kv8_status(int* host_status, cudaStream_t stream) {
  void* addr = nullptr;
  APS_CUDA(cudaGetSymbolAddress(&addr, g_kv8_status));
  APS_CUDA(cudaMemcpyAsync(host_status, addr, sizeof(int), cudaMemcpyDeviceToHost, stream));
  APS_CUDA(cudaStreamSynchronize(stream));
  if (*host_status != 0) APS_CUDA(cudaMemsetAsync(addr, 0, sizeof(int), stream));   // reported once
  return APS_OK;
}

bool kv8_supported(int dtype, int head_size) {
  return dtype_size(dtype) != 0 && (head_size == 32 || head_size == 64 || head_size == 128 || head_size == 256);
}

int check_kv8_cache(const char* op, const Kv8Cache& c, int dtype) {
  APS_REQUIRE(dtype_size(dtype) != 0, APS_ERR_DTYPE, "%s: unsupported dtype %d", op, dtype);
  APS_REQUIRE(c.heads > 0 && c.head_size > 0 && c.block_size > 0 && c.num_blocks >= 0, APS_ERR_SHAPE, "%s: bad sizes", op);
  APS_REQUIRE(c.block_size % 16 == 0 && c.block_size <= 1024, APS_ERR_UNSUPPORTED,
              "%s: block size must be a multiple of 16 up to 1024 (got %d)", op, c.block_size);
  APS_REQUIRE(kv8_supported(dtype, c.head_size), APS_ERR_UNSUPPORTED, "%s: head size %d is not supported", op, c.head_size);
  APS_REQUIRE(c.heads <= 65535, APS_ERR_SHAPE, "%s: too many heads", op);
  APS_REQUIRE(c.block_stride >= (int64_t)c.block_size * c.heads * c.head_size && c.scale_stride >= c.heads, APS_ERR_SHAPE,
              "%s: strides smaller than a block / its scales", op);
  APS_REQUIRE(c.num_blocks <= (int64_t(1) << 31) / c.block_size, APS_ERR_SHAPE, "%s: more than 2^31 slots", op);
  return APS_OK;
}

}  // namespace aps

using namespace aps;

extern "C" int aps_kv8_write(const void* key, const void* value, void* key_cache, void* value_cache, float* key_scale,
                             float* value_scale, const int64_t* slot_mapping, int64_t num_tokens, int num_heads, int head_size,
                             int block_size, int64_t num_blocks, int64_t key_stride, int64_t value_stride, int64_t block_stride,
                             int64_t scale_stride, int dtype, void* stream) {
  const Kv8Cache c{(const uint8_t*)key_cache, (const uint8_t*)value_cache, key_scale, value_scale, num_blocks, block_stride, scale_stride,
                   num_heads, head_size, block_size};
  const int st = check_kv8_cache("kv8_write", c, dtype);
  if (st != APS_OK) return st;
  APS_REQUIRE(num_tokens >= 0 && num_tokens < (int64_t(1) << 31), APS_ERR_SHAPE, "kv8_write: bad number of rows");
  if (num_tokens == 0) return APS_OK;
  APS_REQUIRE(key && value && key_cache && value_cache && key_scale && value_scale && slot_mapping, APS_ERR_NULL_POINTER,
              "kv8_write: null pointer");
  const int64_t row = (int64_t)num_heads * head_size;
  APS_REQUIRE(key_stride >= row && value_stride >= row, APS_ERR_SHAPE, "kv8_write: strides smaller than a row");
  const int es = dtype_size(dtype), vec = 4 * es;
  APS_REQUIRE(aligned_to(key, es) && aligned_to(value, es) && aligned_to(key_cache, 4) && aligned_to(value_cache, 4) &&
                  block_stride % 4 == 0 && aligned_to(key_scale, 4) && aligned_to(value_scale, 4) && aligned_to(slot_mapping, 8),
              APS_ERR_MISALIGNED, "kv8_write: the caches' blocks must begin at multiples of 4 bytes");
  const int by = head_size == 256 ? 2 * vec > 16 ? 16 : 2 * vec : vec;
  const bool aligned = aligned_to(key, by) && aligned_to(value, by) && key_stride * es % by == 0 && value_stride * es % by == 0;
  const WriteArgs a{{key, value}, {(uint8_t*)key_cache, (uint8_t*)value_cache}, {key_scale, value_scale}, slot_mapping, num_tokens,
                    num_blocks, {key_stride, value_stride}, block_stride, scale_stride, num_heads, block_size};
  switch (dtype) {
    case APS_F32: return write_by_head<float>(a, head_size, aligned, (cudaStream_t)stream);
    case APS_F16: return write_by_head<__half>(a, head_size, aligned, (cudaStream_t)stream);
    default: return write_by_head<__nv_bfloat16>(a, head_size, aligned, (cudaStream_t)stream);
  }
}
