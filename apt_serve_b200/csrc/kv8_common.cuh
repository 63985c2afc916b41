// The K/V cache in 8 bits: e4m3 numbers with a scale for each block of tokens and head.
//
// Row element x of block b and head h is held as the e4m3 number nearest to x / s[b][h] (ties to even); NaN and infinities are held
// as NaN.  The writer's scales are powers of two, which costs a number with an exponent of its own nothing (its 4 significant bits
// are the same ones whatever the scale) and makes x / s exact and a block's move to a larger scale a shift of exponents: only what
// falls below the smallest normal number 2^-6 is rounded again.  Readers take any positive scale.
#pragma once

#include "attention_common.cuh"

namespace aps {

// A cache and how it is reached.  Strides of the caches in bytes (= elements), of the scales in elements.
struct Kv8Cache {
  const uint8_t* key; const uint8_t* value;
  const float* key_scale; const float* value_scale;
  int64_t num_blocks, block_stride, scale_stride;
  int heads, head_size, block_size;
};

// One attention call.  Row t of the query belongs to the request r with starts[r] <= t < starts[r + 1] (starts == NULL: t itself);
// the rows of a request are the last of its seq_lens[r] tokens, each attends to the tokens up to itself.
struct Kv8Call {
  void* out; const void* query;
  Kv8Cache cache;
  const int32_t* tables; const int32_t* starts; const int32_t* seq_lens;
  int batch, max_blocks, max_rows;   // max_rows: most rows of a request; those of one that has more are left as they are
  int64_t rows, query_stride, out_stride;
  float scale;
  int dtype;
};

constexpr float kE4m3Max = 448.f;

// The two e4m3 numbers in the low 16 bits as fp16 (exact).
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t codes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(codes));
  return r;
}
// The four of a word, the halves taken apart by the conversion itself.
__device__ __forceinline__ void e4m3x4_to_f16x4(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(codes));
}
// Four numbers of a word as floats.
__device__ __forceinline__ void e4m3x4_to_float(uint32_t codes, float* f) {
  uint32_t lo, hi;
  e4m3x4_to_f16x4(codes, lo, hi);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
}
// To the nearest, ties to even; beyond 448 to 448, NaN to 0x7f.
__device__ __forceinline__ uint16_t float2_to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t float4_to_e4m3x4(const float* f) {
  return (uint32_t)float2_to_e4m3x2(f[0], f[1]) | (uint32_t)float2_to_e4m3x2(f[2], f[3]) << 16;
}
__device__ __forceinline__ uint16_t f16x2_to_e4m3x2(uint32_t halves) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(halves));
  return r;
}
// The smallest power of two s >= 2^-118 with top <= 448 s (448 = 1.75 * 2^8; top finite and not negative).
__device__ __forceinline__ float e4m3_scale(float top) {
  const uint32_t u = __float_as_uint(top);
  const int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);   // biased; a subnormal top gives the least scale
  return __uint_as_float((uint32_t)max(e, 127 - 118) << 23);
}

// Where the parts of rows whose tokens are cut go: [row][head][split], and the header of the scratch (PlanWord).
struct Kv8Parts {
  int* plan;
  float2* ml;                // maximum of the scores (log2) and sum of the weights relative to it; nothing attended: (-infinity, 0), scores
                             // that are all NaN: (-infinity, NaN)
  float* acc;                // weighted values, relative to that maximum
  int splits;                // 1: the output is written directly
  float scale_log2;
};

// The request of query row t, and how many tokens the row attends to (none: a zero row).  False: the row belongs to no request, or
// comes behind the max_rows first ones of its own.
__device__ __forceinline__ bool kv8_find_row(const Kv8Call& c, int64_t t, int& req, int& keys) {
  if (c.starts == nullptr) {
    req = (int)t;
    keys = max(0, min(c.seq_lens[req], c.max_blocks * c.cache.block_size));
    return true;
  }
  if (t < c.starts[0] || t >= c.starts[c.batch]) return false;
  int lo = 0, hi = c.batch;   // starts[lo] <= t < starts[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (c.starts[mid] <= t) lo = mid; else hi = mid;
  }
  req = lo;
  if (t - c.starts[req] >= c.max_rows) return false;
  const int ctx = max(0, min(c.seq_lens[req], c.max_blocks * c.cache.block_size));
  keys = max(0, ctx - c.starts[req + 1] + (int)t + 1);
  return true;
}

// x / n by the high word of x * ceil(2^32 / n), n the blocks' size in groups of 16 tokens (up to 64): exact for x below 2^26.  0: n is 1.
inline uint32_t kv8_blocks_magic(int block_size) {
  const uint32_t n = block_size / 16;
  return n == 1 ? 0u : (uint32_t)(((uint64_t(1) << 32) + n - 1) / n);
}

// Up to 16 query rows per request (kv8_stream.cu).
bool kv8_stream_takes(const Kv8Call& c);
int kv8_stream_splits(const Kv8Call& c);
int launch_kv8_stream(const Kv8Call& c, const Kv8Parts& parts, cudaStream_t stream);

// Query rows by tiles of 128 on the tensor cores (kv8_prefix.cu).
bool kv8_tiles_take(const Kv8Call& c);
int kv8_tile_splits(const Kv8Call& c);
int kv8_tile_splits(const Kv8Call& c, int tiles);   // with one or two row tiles per CTA
int launch_kv8_tiles(const Kv8Call& c, const Kv8Parts& parts, cudaStream_t stream);

bool kv8_supported(int dtype, int head_size);
int check_kv8_cache(const char* op, const Kv8Cache& c, int dtype);
int read_kv8_status(int* host_status, cudaStream_t stream);   // kv8_write.cu

}  // namespace aps
