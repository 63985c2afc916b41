// Rows of K and V into the 8-bit cache (kv8_common.cuh).
//
// Stands beside aps_reshape_and_cache, with the same slots: slot / BS is the block, slot % BS the row in it.  All rows of a call that
// go to one block are taken together, whatever their order in the mapping (of two rows for one slot the later one stays).  If the
// block's first slot is among them the block starts anew: its scale is that of the new rows, its other rows are left as they are.
// Otherwise the block's scale becomes the larger of the old one and the new rows', and, where it grows, the block's other rows are
// rounded to it.
//
// A warp takes one head of one plane of a block: its rows in registers (16 rows of 16-byte pieces in flight at once), the largest
// element by shuffles, then the codes.  Which rows belong together:
//   few rows    every row's CTAs look through the whole mapping; those of a block's first row do the block (one launch)
//   many rows   runs of neighbouring rows in neighbouring slots of one block are listed first (prompts are nothing else), with how many
//               such runs a block has; a block that has one is done from its run, others by looking through the mapping
// What bounds it: bytes, (element size + 1) for each element of prompts' rows; launch and three round trips (mapping; scale and
// rows; the block's other rows) for few single tokens, rounds of CTAs that each look through the mapping for many: 256 tokens of 40 x 128
// are 2560 CTAs, 592 at a time, 15 us.  24 OPT-13B prompts in fp16 (592 MB) 126 us, 72 % of the measured copy rate: the loads' latency at
// the 32 warps an SM that registers leave room for, 4 KB each in flight (47 % of its warps, 53 % of the issue slots).
// Spills, at 64 registers: rows of 128 in the kernels for runs 84 - 88 bytes, with blocks of more than 16 rows 208 - 224; rows of 256 up to
// 728; fp32, at 128 registers, 4 - 88.
#include "kv8_common.cuh"

#include <type_traits>

namespace aps {
namespace {

constexpr int kThreads = 256;

__device__ int g_kv8_status = 0;   // a slot past the cache has been met since this was read last

// Whether there has been a write on the current device (of which a captured one may be replayed at any time): reading the status is a
// copy to the host, which callers without an 8-bit cache are spared.
bool* written_here() {
  static bool written[64] = {false};
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64 ? &written[dev] : nullptr;
}

struct WriteArgs {
  const void *key, *value;
  uint8_t *key_cache, *value_cache;
  float *key_scale, *value_scale;
  const int64_t* slots;
  int64_t tokens, num_blocks, key_stride, value_stride, block_stride, scale_stride;
  int heads, block_size;
};

template <typename T, int D> struct RowCfg {
  static constexpr int kPer = 16 / sizeof(T) < D / 4 ? 16 / sizeof(T) : D / 4;   // elements per lane: 16 bytes
  static constexpr int kLanes = D / kPer > 32 ? 32 : D / kPer;                   // lanes per row
  static constexpr int kParts = D / (kPer * kLanes);                             // pieces per lane (fp32 rows of 256)
  static constexpr int kRows = 32 / kLanes;                                      // rows a warp has at a time
  static constexpr int kLoads = 16 / kRows * kParts;                             // pieces of 16 rows
};

// CTAs per SM: a lane's share of 16 rows of 128 takes 32 registers, in fp32 64.
template <typename T> __host__ __device__ constexpr int run_ctas() { return sizeof(T) == 2 ? 4 : 2; }

template <typename T, int N> struct alignas(N * sizeof(T)) Pack { T x[N]; };

// The largest magnitude of what has been seen (`some`, pairs of 16-bit numbers or a float) and of p; NaN does not count.
template <typename T> struct Magnitude { using Type = float; };
template <> struct Magnitude<__half> { using Type = __half2; };
template <> struct Magnitude<__nv_bfloat16> { using Type = __nv_bfloat162; };
template <typename T, int N>
__device__ __forceinline__ typename Magnitude<T>::Type magnitude(const Pack<T, N>& p, typename Magnitude<T>::Type some) {
  if constexpr (sizeof(T) == 2) {
    const auto* x = reinterpret_cast<const typename Magnitude<T>::Type*>(&p);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) some = __hmax2(some, __habs2(x[i]));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) some = fmaxf(some, fabsf(p.x[i]));
  }
  return some;
}
__device__ __forceinline__ float magnitude_value(float some) { return some; }
__device__ __forceinline__ float magnitude_value(__half2 some) { return fmaxf(__low2float(some), __high2float(some)); }
__device__ __forceinline__ float magnitude_value(__nv_bfloat162 some) { return fmaxf(__low2float(some), __high2float(some)); }

// N finite elements times a power of two as e4m3 numbers.
template <typename T, int N>
__device__ __forceinline__ void quantise(const Pack<T, N>& p, float by, uint32_t* out) {
#pragma unroll
  for (int q = 0; q < N / 4; ++q) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = Elem<T>::to_float(p.x[4 * q + e]) * by;
    out[q] = float4_to_e4m3x4(y);
  }
}
// The same in fp16, by a normal number: what the product loses there is below 2^-24, and zero in e4m3 anyway.
template <int N>
__device__ __forceinline__ void quantise_half(const Pack<__half, N>& p, __half2 by, uint32_t* out) {
  const __half2* x = reinterpret_cast<const __half2*>(&p);
#pragma unroll
  for (int q = 0; q < N / 4; ++q) {
    const __half2 a = __hmul2(x[2 * q], by), b = __hmul2(x[2 * q + 1], by);
    out[q] = (uint32_t)f16x2_to_e4m3x2(*reinterpret_cast<const uint32_t*>(&a)) |
             (uint32_t)f16x2_to_e4m3x2(*reinterpret_cast<const uint32_t*>(&b)) << 16;
  }
}

// The rows that a block gets: n of them, either row + k to slot + k, or by two lists, the slots that get one and each slot's row.
struct BlockRows {
  uint32_t block;
  int n, row, slot;
  const int* slots;    // NULL: neighbours
  const int* token;
  __device__ __forceinline__ int row_of(int k) const { return slots == nullptr ? row + k : token[slots[k]]; }
  __device__ __forceinline__ int slot_of(int k) const { return slots == nullptr ? slot + k : slots[k]; }
  __device__ __forceinline__ bool taken(int o) const { return slots == nullptr ? o >= slot && o < slot + n : token[o] >= 0; }
};

// One head of one plane of a block, by one warp: any rows, any values, element by element.
template <typename T, int D>
__device__ __forceinline__ void write_any_head(const WriteArgs& a, int plane, int head, const BlockRows& b, int lane) {
  constexpr int kPer = D / 32;   // elements per lane
  const T* rows = static_cast<const T*>(plane ? a.value : a.key) + (int64_t)head * D + lane * kPer;
  uint8_t* held = (plane ? a.value_cache : a.key_cache) + (int64_t)b.block * a.block_stride + (int64_t)head * D + lane * kPer;
  const int64_t step = plane ? a.value_stride : a.key_stride, held_row = (int64_t)a.heads * D;
  float* scale_at = (plane ? a.value_scale : a.key_scale) + (int64_t)b.block * a.scale_stride + head;
  const float old = *scale_at;
  const bool anew = b.taken(0);
  float top = 0.f;
#pragma unroll 1
  for (int k = 0; k < b.n; ++k) {
    const T* x = rows + b.row_of(k) * step;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const float y = fabsf(Elem<T>::to_float(x[e]));
      top = fmaxf(top, y <= 3.402823466e38f ? y : 0.f);   // NaN and infinities have no part in it
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float need = e4m3_scale(top), s = anew ? need : fmaxf(old, need), ratio = old / s;
#pragma unroll 1
  for (int k = 0; k < b.n; ++k) {
    const T* x = rows + b.row_of(k) * step;
    uint8_t* to = held + b.slot_of(k) * held_row;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const float z = Elem<T>::to_float(x[e]);
      to[e] = (uint8_t)float2_to_e4m3x2(fabsf(z) <= 3.402823466e38f ? z / s : __int_as_float(0x7fc00000), 0.f);
    }
  }
  if (!anew && s != old) {   // the block's other rows
#pragma unroll 1
    for (int o = 0; o < a.block_size; ++o) {
      if (b.taken(o)) continue;
      uint8_t* to = held + o * held_row;
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const uint32_t h = e4m3x2_to_f16x2(to[e]);
        to[e] = (uint8_t)float2_to_e4m3x2(__half2float(__ushort_as_half((unsigned short)h)) * ratio, 0.f);
      }
    }
  }
  if (lane == 0 && s != old) *scale_at = s;
}

// 16 rows at a time in registers, 16 bytes of each, blocks of any size (their rows come a second time, from L2), the block's other rows
// rounded to a larger scale; no infinities, a scale that is a power of two.  False: nothing has been written.
template <typename T, int D, bool kAligned>
__device__ __forceinline__ bool write_rows(const WriteArgs& a, int plane, int head, const BlockRows& b, int lane) {
  using C = RowCfg<T, D>;
  using P = Pack<T, C::kPer>;
  constexpr int kWords = C::kPer / 4;
  if (!kAligned || C::kParts > 1) return false;
  const int at = lane / C::kLanes, column = lane % C::kLanes * C::kPer;
  const T* rows = static_cast<const T*>(plane ? a.value : a.key) + (int64_t)head * D + column;
  const int64_t step = plane ? a.value_stride : a.key_stride;
  float* scale_at = (plane ? a.value_scale : a.key_scale) + (int64_t)b.block * a.scale_stride + head;
  const float old = *scale_at;
  P x[C::kLoads];
  auto load = [&](int from) {
#pragma unroll
    for (int i = 0; i < C::kLoads; ++i) {
      const int k = from + i * C::kRows + at;
      if (from + i * C::kRows < b.n) x[i] = *reinterpret_cast<const P*>(rows + (int64_t)(k < b.n ? b.row_of(k) : b.row_of(0)) * step);   // a row twice is no harm
    }
  };
  typename Magnitude<T>::Type some{};
  const int last = (b.n - 1) / 16 * 16;
#pragma unroll 1
  for (int from = 0; from <= last; from += 16) {
    load(from);
#pragma unroll
    for (int i = 0; i < C::kLoads; ++i)
      if (from + i * C::kRows < b.n) some = magnitude<T, C::kPer>(x[i], some);
  }
  // numbers that are not negative are in the order of their bits
  const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(magnitude_value(some))));
  const bool anew = b.taken(0);
  const float need = e4m3_scale(top), s = anew ? need : fmaxf(old, need), by = 1.f / s;
  if (!(top <= 3.402823466e38f) || (__float_as_uint(s) & 0x7fffffu) != 0) return false;
  uint8_t* held = (plane ? a.value_cache : a.key_cache) + (int64_t)b.block * a.block_stride + (int64_t)head * D + column;
  const int64_t held_row = (int64_t)a.heads * D;
  const bool in_half = std::is_same<T, __half>::value && by >= 6.103515625e-05f && by <= 32768.f;
#pragma unroll 1
  for (int from = last; from >= 0; from -= 16) {   // the last 16 are still there
    if (from < last) load(from);
#pragma unroll
    for (int i = 0; i < C::kLoads; ++i) {
      const int k = from + i * C::kRows + at;
      if (k < b.n) {
        uint32_t w[kWords];
        if constexpr (std::is_same<T, __half>::value) {
          if (in_half) quantise_half<C::kPer>(x[i], __float2half2_rn(by), w);
          else quantise<T, C::kPer>(x[i], by, w);
        } else {
          quantise<T, C::kPer>(x[i], by, w);
        }
        uint32_t* to = reinterpret_cast<uint32_t*>(held + b.slot_of(k) * held_row);
        if constexpr (kWords == 2) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
        else to[0] = w[0];
      }
    }
  }
  if (!anew && s != old) {   // the block's other rows, 16 slots in one round trip
    const float ratio = old / s;
#pragma unroll 1
    for (int from = 0; from < a.block_size; from += 16) {
      uint32_t w[C::kLoads][kWords];
#pragma unroll
      for (int i = 0; i < C::kLoads; ++i) {
        const uint32_t* p = reinterpret_cast<const uint32_t*>(held + (from + i * C::kRows + at) * held_row);
#pragma unroll
        for (int q = 0; q < kWords; ++q) w[i][q] = p[q];
      }
#pragma unroll
      for (int i = 0; i < C::kLoads; ++i) {
        const int o = from + i * C::kRows + at;
        if (b.taken(o)) continue;
        uint32_t* to = reinterpret_cast<uint32_t*>(held + o * held_row);
#pragma unroll
        for (int q = 0; q < kWords; ++q) {
          float y[4];
          e4m3x4_to_float(w[i][q], y);
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] *= ratio;
          to[q] = float4_to_e4m3x4(y);
        }
      }
    }
  }
  if (lane == 0 && s != old) *scale_at = s;
  return true;
}

// For what almost all blocks get: up to 16 rows, 16 bytes at a time, all of them in registers; no infinities, a scale that is a power of
// two, no other rows to be rounded to it.  False: nothing has been written, one of the forms above has to do it (after the kernel's other
// heads: between them its registers would be this one's; in one function with the form above 24 OPT-13B prompts took 158 us, so 126).
// Offset: of a row in the block; 32 bits where the block has 16 rows (with 64, and one call for both forms, they took 135).
template <typename T, int D, bool kAligned, typename Offset>
__device__ __forceinline__ bool write_head(const WriteArgs& a, int plane, int head, const BlockRows& b, int lane) {
  using C = RowCfg<T, D>;
  using P = Pack<T, C::kPer>;
  constexpr int kWords = C::kPer / 4;
  if (!kAligned || C::kParts > 1 || b.n > 16) return false;
  const int at = lane / C::kLanes, column = lane % C::kLanes * C::kPer;
  const T* rows = static_cast<const T*>(plane ? a.value : a.key) + (int64_t)head * D + column;
  const int64_t step = plane ? a.value_stride : a.key_stride;
  float* scale_at = (plane ? a.value_scale : a.key_scale) + (int64_t)b.block * a.scale_stride + head;
  const float old = *scale_at;
  P x[C::kLoads];
#pragma unroll
  for (int i = 0; i < C::kLoads; ++i) {
    const int k = i * C::kRows + at;
    if (i * C::kRows < b.n) {
      const P* p = reinterpret_cast<const P*>(rows + (int64_t)(k < b.n ? b.row_of(k) : b.row_of(0)) * step);   // a row twice is no harm
      x[i] = *p;
    }
  }
  typename Magnitude<T>::Type some{};
#pragma unroll
  for (int i = 0; i < C::kLoads; ++i)
    if (i * C::kRows < b.n) some = magnitude<T, C::kPer>(x[i], some);
  // numbers that are not negative are in the order of their bits
  const float top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(magnitude_value(some))));
  const bool anew = b.taken(0);
  const float need = e4m3_scale(top), s = anew ? need : fmaxf(old, need), by = 1.f / s;
  if (!(top <= 3.402823466e38f) || (__float_as_uint(s) & 0x7fffffu) != 0 || (!anew && s != old)) return false;
  uint8_t* held = (plane ? a.value_cache : a.key_cache) + (int64_t)b.block * a.block_stride + (int64_t)head * D + column;
  const Offset held_row = (Offset)a.heads * D;
  const bool in_half = std::is_same<T, __half>::value && by >= 6.103515625e-05f && by <= 32768.f;
#pragma unroll
  for (int i = 0; i < C::kLoads; ++i) {
    const int k = i * C::kRows + at;
    if (k < b.n) {
      uint32_t w[kWords];
      if constexpr (std::is_same<T, __half>::value) {
        if (in_half) quantise_half<C::kPer>(x[i], __float2half2_rn(by), w);
        else quantise<T, C::kPer>(x[i], by, w);
      } else {
        quantise<T, C::kPer>(x[i], by, w);
      }
      uint32_t* to = reinterpret_cast<uint32_t*>(held + b.slot_of(k) * held_row);
      if constexpr (kWords == 2) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
      else to[0] = w[0];
    }
  }
  if (lane == 0 && s != old) *scale_at = s;
  return true;
}

// The rows of a block by slot, as a list: slot and row, the slots in order.
__device__ __forceinline__ int list_rows(const int* token, int* slots, int block_size, int lane) {
  int n = 0;
  for (int o = lane; o < block_size + lane; o += 32) {
    const bool has = o < block_size && token[o] >= 0;
    const uint32_t who = __ballot_sync(0xffffffffu, has);
    if (has) slots[n + __popc(who & ((1u << lane) - 1))] = o;
    n += __popc(who);
  }
  return n;
}

// ---- few rows: one CTA per (row, some heads); the CTAs of the first row of a block do the block ----
template <typename T, int D, bool kAligned>
__global__ void __launch_bounds__(kThreads, run_ctas<T>())
kv8_write_kernel(const WriteArgs a) {
  extern __shared__ int token[];   // [block_size] rows by slot, [block_size] slots that get one
  __shared__ int s_later, s_n;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  chain_wait();
  chain_next();
  const int t = blockIdx.x, tokens = (int)a.tokens;
  const int64_t slot = a.slots[t], before = t > 0 ? a.slots[t - 1] : -1;
  if (slot < 0) return;
  if (slot >= a.num_blocks * a.block_size) {
    if (tid == 0) g_kv8_status = kStatusBadIndex;
    return;
  }
  const uint32_t block = (uint32_t)slot / (uint32_t)a.block_size;
  const int64_t first = (int64_t)block * a.block_size;
  auto same = [&](int64_t other) { return other >= first && other < first + a.block_size; };
  if (same(before)) return;
  for (int o = tid; o < a.block_size; o += kThreads) token[o] = -1;
  if (tid == 0) s_later = 0;
  __syncthreads();
  for (int i = tid; i < tokens; i += kThreads) {
    const int64_t other = a.slots[i];
    if (!same(other)) continue;
    if (i < t) s_later = 1;
    atomicMax(&token[other - first], i);
  }
  __syncthreads();
  if (s_later) return;
  int* slots = token + a.block_size;
  if (warp == 0) {
    const int n = list_rows(token, slots, a.block_size, lane);
    if (lane == 0) s_n = n;
  }
  __syncthreads();
  const int u = blockIdx.y * (kThreads / 32) + warp;
  if (u >= 2 * a.heads) return;
  const int plane = u >= a.heads, head = plane ? u - a.heads : u;
  const BlockRows b{block, s_n, 0, 0, slots, token};
  if (!write_head<T, D, kAligned, int64_t>(a, plane, head, b, lane) && !write_rows<T, D, kAligned>(a, plane, head, b, lane))
    write_any_head<T, D>(a, plane, head, b, lane);
}

// ---- many rows ----
// Runs: neighbouring rows of one block in neighbouring slots.  blocks: how many runs a block has, and the last row of its run;
// list: first row and slot of each run; number: of runs.
struct Runs { int2* blocks; int* number; int2* list; };

__global__ void __launch_bounds__(256)
kv8_runs_kernel(const WriteArgs a, const Runs r) {
  chain_wait();
  chain_next();
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= a.tokens) return;
  const int64_t slot = a.slots[t];
  if (slot < 0) return;
  if (slot >= a.num_blocks * a.block_size) { g_kv8_status = kStatusBadIndex; return; }
  const uint32_t block = (uint32_t)slot / (uint32_t)a.block_size;
  const bool begins = slot == (int64_t)block * a.block_size, ends = slot + 1 == (int64_t)(block + 1) * a.block_size;
  if (begins || t == 0 || a.slots[t - 1] != slot - 1) {
    atomicAdd(&r.blocks[block].x, 1);
    r.list[atomicAdd(r.number, 1)] = make_int2((int)t, (int)slot);
  }
  if (ends || t == a.tokens - 1 || a.slots[t + 1] != slot + 1) r.blocks[block].y = (int)t;
}

// Every warp for itself: one head of one plane of one run after the other.
// kShort: blocks of 16 rows.
template <typename T, int D, bool kAligned, bool kShort>
__global__ void __launch_bounds__(kThreads, run_ctas<T>())
kv8_write_runs_kernel(const WriteArgs a, const Runs r) {
  extern __shared__ int tokens[];   // [warps][2 * block_size], for blocks of several runs
  chain_wait();
  chain_next();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, which = blockIdx.y * (kThreads / 32) + warp;
  if (which >= 2 * a.heads) return;
  const int plane = which >= a.heads, head = plane ? which - a.heads : which, number = *r.number, step = gridDim.x;
  for (int at = blockIdx.x; at < number; at += 32 * step) {
    uint32_t left = 0;   // of 32 runs, those for the other forms
    // what a run is about comes in two round trips: the next one's block and the one's after that are on their way meanwhile
    auto run_at = [&](int k) { return k < 32 && at + k * step < number ? r.list[at + k * step] : make_int2(0, 0); };
    auto block_of = [&](int2 run) { return (uint32_t)run.y / (uint32_t)a.block_size; };
    int2 now = run_at(0), then = run_at(1), info = r.blocks[block_of(now)];
    for (int k = 0; k < 32 && at + k * step < number; ++k) {
      const int2 after = run_at(k + 2), next_info = r.blocks[block_of(then)];
      const uint32_t block = block_of(now);
      const int from = now.y - (int)(block * (uint32_t)a.block_size);
      if constexpr (kShort) {
        if (info.x != 1 || !write_head<T, D, kAligned, int>(a, plane, head, BlockRows{block, info.y - now.x + 1, now.x, from, nullptr, nullptr}, lane))
          left |= 1u << k;
      } else {
        if (info.x != 1 || !write_rows<T, D, kAligned>(a, plane, head, BlockRows{block, info.y - now.x + 1, now.x, from, nullptr, nullptr}, lane))
          left |= 1u << k;
      }
      now = then; then = after; info = next_info;
    }
    for (; left != 0; left &= left - 1) {
      const int2 now = r.list[at + (__ffs(left) - 1) * step];
      const uint32_t block = (uint32_t)now.y / (uint32_t)a.block_size;
      const int2 info = r.blocks[block];
      BlockRows b{block, info.y - now.x + 1, now.x, now.y - (int)(block * (uint32_t)a.block_size), nullptr, nullptr};
      if (info.x != 1) {
        int *token = tokens + warp * 2 * a.block_size, *slots = token + a.block_size;
        const int64_t first = (int64_t)block * a.block_size;
        __syncwarp();
        for (int o = lane; o < a.block_size; o += 32) token[o] = -1;
        __syncwarp();
        bool mine = true;   // the first run of the block does it
        for (int64_t k = lane; k < a.tokens; k += 32) {
          const int64_t other = a.slots[k];
          if (other < first || other >= first + a.block_size) continue;
          mine = mine && k >= now.x;
          atomicMax(&token[other - first], (int)k);
        }
        if (!__all_sync(0xffffffffu, mine)) continue;
        b = BlockRows{block, list_rows(token, slots, a.block_size, lane), 0, 0, slots, token};
        __syncwarp();
      }
      write_any_head<T, D>(a, plane, head, b, lane);
    }
  }
}

// Up to so many rows every CTA looks through the mapping.
constexpr int64_t kScanRows = 1024;

size_t write_scratch(int64_t tokens, int64_t blocks) {
  return tokens <= kScanRows ? 0 : (kPlanWords + 2) * sizeof(int) + ((size_t)blocks + (size_t)tokens) * sizeof(int2);
}

template <typename T, int D, bool kAligned>
int launch_write(const WriteArgs& a, void* workspace, cudaStream_t stream) {
  const int slices = (2 * a.heads + kThreads / 32 - 1) / (kThreads / 32);
  if (a.tokens <= kScanRows) {
    return launch_chained("kv8_write_kernel", kv8_write_kernel<T, D, kAligned>, dim3((unsigned)a.tokens, slices), kThreads,
                          2 * a.block_size * sizeof(int), stream, a);
  }
  int* base = static_cast<int*>(workspace) + kPlanWords;   // the attention calls' header stays as it is
  int2* blocks = reinterpret_cast<int2*>(base + 2);
  const Runs r{blocks, base, blocks + a.num_blocks};
  APS_CUDA(cudaMemsetAsync(base, 0, 2 * sizeof(int) + (size_t)a.num_blocks * sizeof(int2), stream));
  int st = launch_chained("kv8_runs_kernel", kv8_runs_kernel, (unsigned)((a.tokens + 255) / 256), 256, 0, stream, a, r);
  if (st != APS_OK) return st;
  const size_t smem = (size_t)kThreads / 32 * 2 * a.block_size * sizeof(int);
  auto kernel = a.block_size == 16 ? kv8_write_runs_kernel<T, D, kAligned, true> : kv8_write_runs_kernel<T, D, kAligned, false>;
  if (smem > 48 * 1024) APS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  int64_t x = (int64_t)sm_count() * run_ctas<T>() / slices;   // and no few more that would run alone in the end
  x = x < 1 ? 1 : x > a.tokens ? a.tokens : x;
  return launch_chained("kv8_write_runs_kernel", kernel, dim3((unsigned)x, slices), kThreads, smem, stream, a, r);
}

template <typename T>
int write_by_head(const WriteArgs& a, int head_size, bool aligned, void* ws, cudaStream_t stream) {
  switch (head_size) {
    case 32: return aligned ? launch_write<T, 32, true>(a, ws, stream) : launch_write<T, 32, false>(a, ws, stream);
    case 64: return aligned ? launch_write<T, 64, true>(a, ws, stream) : launch_write<T, 64, false>(a, ws, stream);
    case 128: return aligned ? launch_write<T, 128, true>(a, ws, stream) : launch_write<T, 128, false>(a, ws, stream);
    default: return aligned ? launch_write<T, 256, true>(a, ws, stream) : launch_write<T, 256, false>(a, ws, stream);
  }
}

}  // namespace

int read_kv8_status(int* host_status, cudaStream_t stream) {
  const bool* written = written_here();
  if (written != nullptr && !*written) {
    *host_status = 0;
    return APS_OK;
  }
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

extern "C" size_t aps_kv8_write_workspace_bytes(int64_t num_tokens, int64_t num_blocks) {
  return num_tokens <= 0 || num_blocks <= 0 ? 0 : write_scratch(num_tokens, num_blocks);
}

extern "C" int aps_kv8_write(const void* key, const void* value, void* key_cache, void* value_cache, float* key_scale,
                             float* value_scale, const int64_t* slot_mapping, int64_t num_tokens, int num_heads, int head_size,
                             int block_size, int64_t num_blocks, int64_t key_stride, int64_t value_stride, int64_t block_stride,
                             int64_t scale_stride, void* workspace, size_t workspace_bytes, int dtype, void* stream) {
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
  const int es = dtype_size(dtype);
  APS_REQUIRE(aligned_to(key, es) && aligned_to(value, es) && aligned_to(key_cache, 4) && aligned_to(value_cache, 4) &&
                  block_stride % 4 == 0 && aligned_to(key_scale, 4) && aligned_to(value_scale, 4) && aligned_to(slot_mapping, 8),
              APS_ERR_MISALIGNED, "kv8_write: the caches' blocks must begin at multiples of 4 bytes");
  const size_t need = write_scratch(num_tokens, num_blocks);
  APS_REQUIRE(need == 0 || (workspace != nullptr && aligned_to(workspace, 256) && workspace_bytes >= need), APS_ERR_WORKSPACE,
              "kv8_write: workspace must be 256-byte aligned and hold %zu bytes (got %zu)", need, workspace_bytes);
  if (bool* written = written_here()) *written = true;
  const bool aligned = aligned_to(key, 16) && aligned_to(value, 16) && key_stride * es % 16 == 0 && value_stride * es % 16 == 0 &&
                       aligned_to(key_cache, 8) && aligned_to(value_cache, 8) && block_stride % 8 == 0;
  const WriteArgs a{key, value, (uint8_t*)key_cache, (uint8_t*)value_cache, key_scale, value_scale, slot_mapping, num_tokens,
                    num_blocks, key_stride, value_stride, block_stride, scale_stride, num_heads, block_size};
  switch (dtype) {
    case APS_F32: return write_by_head<float>(a, head_size, aligned, workspace, (cudaStream_t)stream);
    case APS_F16: return write_by_head<__half>(a, head_size, aligned, workspace, (cudaStream_t)stream);
    default: return write_by_head<__nv_bfloat16>(a, head_size, aligned, workspace, (cudaStream_t)stream);
  }
}
