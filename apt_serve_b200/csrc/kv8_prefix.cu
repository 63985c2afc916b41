// Several query rows per request over the 8-bit cache (kv8_common.cuh), fp16 / bf16 queries, head sizes 64 and 128.
//
// One CTA per (128 query rows of a request, head, part of the tokens), two CTAs per SM; requests of more than 128 rows: one CTA per SM with
// two row tiles, which share the keys and values that it turns into fp16.  Key tiles of 64 tokens up to the diagonal:
//   four warps turn the tile's codes into fp16 on their way from the cache to shared memory (every e4m3 number is an fp16 number)
//   S = Q K^T   tcgen05, M = 128 rows, N = 64 tokens, both operands K-major in shared memory, S in one of two buffers of tensor memory
//   a thread per query row turns its row of S into weights, in fp16 over S
//   O += P V    tcgen05, A = P from tensor memory, B = V MN-major
// The scales never meet a rounded number: a block's key scale multiplies the row's fp32 scores, its value scale the fp32 weight before
// that is rounded to fp16 (11 bits; the cache itself holds 4).  The two have running references of their own: m, the maximum of the
// scores (log2), for the sum of the weights l, and R, the maximum of score + log2(value scale), for the weights that meet V: so a block
// of small values that has all the weight fills fp16's range like any other.  O stays in tensor memory and is rescaled only when R has
// grown by more than 2^8.  The output is O 2^(R - m) / l.
// The weights go into P V as one fp16 term.  Prompts' own attention (prefill_attention.cu) adds the rounded rest as a second one, because
// its rows are exact and the weights' 2^-11 shows in its outputs; here every row has been rounded to 4 bits, 2.6e-2 of it, beside which
// outputs at 2.8e-4 of those over the codes, where 2.1e-4 are the rounding of fp16 outputs (bf16 1.66e-3 and 1.65e-3), show next to nothing.
// The second term would double P V's instructions and took a fifth of the time there.
// bf16 queries become fp16 with a power of two for each row, which leaves 2^-40 of the row's largest element.
//
// Measured on one B200: 500 new tokens each of six OPT-13B requests behind 1000 (83 GFLOP) 178 us, 2048 of a 16 001-token OPT-1.3B document
// (251 GFLOP) 514 (bf16 183 and 516).  A pair of row tiles takes 1900 cycles a key tile (D = 64; 128: 2400) where its exponentials take
// 1024 (16 a cycle and SM), the products 640 (D = 64) to 1280: a softmax warp is busy for 1700 of them, 1100 in the exponentials, which
// both tiles take at the same time; issue slots 46 %, special function unit 57 % (document; chunks 32 and 29 %).
// Registers: two CTAs an SM leave the one-tile form 96, of which 48 - 52 bytes are spilled, in bf16 with D = 128 448; the two-tile form
// spills 52 bytes there and none elsewhere.
// Tried, chunks / document, us: key tiles of 128 with one S 270 / 785 (183 / 517 without, before the copies were tile by tile); beside
// 185 / 528: the second row tile held back by half a turn 196 / 563, two threads per row 200 / 569, a quarter of the exponentials as
// polynomials 194 / 578, three stages of K and V 191 / 544, one row tile per CTA for long requests too 205 / 561; a warp for the products
// of each row tile, with and without that half turn, 180 - 184 / 523; with D = 64 the queries in tensor memory 515 (514 from shared memory).
#include "kv8_common.cuh"
#include "sm100.cuh"

#include <type_traits>

namespace aps {
namespace {

constexpr int kRows = 128, kCopyWarps = 4, kSoftWarp = 1 + kCopyWarps;
constexpr int kKeys = 64, kGroups = kKeys / 16;
constexpr float kSlack = 8.f;   // log2 of how much R may have grown before O is rescaled
constexpr float kUp = 7.f;      // log2 of what the weights are kept at: 2^15 at most
constexpr int kStatusTileWait = 6;

// kTiles: tiles of 128 rows that share the CTA's keys and values.
template <int kTiles>
struct Aux {
  // key tile j: entry j & 1, phase j >> 1
  uint64_t q_full, k_full[2], v_full[2], k_empty[2], v_empty[2], s_full[kTiles][2], p_full[kTiles][2], o_done[kTiles][2];
  uint64_t scales_full[4];        // entry j & 3, phase j >> 2: written again only after the weights of tile j + 1
  float2 scales[4][kKeys / 16];   // key scale, log2 of the value scale
  uint32_t tmem_base;
  int abort_flag;
};

__device__ __forceinline__ void mma_tmem_a(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "mov.b64 db, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
// tmem_ld32's registers may be read behind this.
__device__ __forceinline__ void tmem_ld_wait32(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
      : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
      "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
      "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
      "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
      :: "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Not moved behind the waits that follow it.
__device__ __forceinline__ uint4 ld_ahead(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// Two at a time.
__device__ __forceinline__ float2 fma2(float2 a, float b, float c) {
  uint64_t x, y, z;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %1};" : "=l"(y) : "f"(b));
  asm("mov.b64 %0, {%1, %1};" : "=l"(z) : "f"(c));
  asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(x) : "l"(y), "l"(z));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a.x), "=f"(a.y) : "l"(x));
  return a;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t x, y;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(y));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a.x), "=f"(a.y) : "l"(x));
  return a;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void st_shared16(uint32_t addr, const uint32_t* w) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
}

template <int D, int kTiles> __host__ __device__ constexpr size_t tile_smem() { return 1024 + (size_t)(kTiles * kRows + 4 * kKeys) * D * 2; }

// The CTAs' rows, those with the most tokens first: which of the batch * blocks pairs of a request and kTall of its rows (its last ones first)
// comes at place `rank`.  Ragged batches end together then: six chunks of 424 ... 670 rows 181 us in the order of the requests, 177 in
// this one; 2048 rows of a document (the last ones first for all heads, not for each) 527 and 514.
// More than kSorted pairs keep the requests' order: what the last ones are late by is little of the whole.
constexpr int kSorted = 256;

template <int kTall>
__device__ __forceinline__ int longest_first(const Kv8Call& c, int blocks, int rank) {
  const int pairs = c.batch * blocks;
  if (pairs > kSorted) return rank;
  __shared__ int s_tokens[kSorted], s_pair;
  for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
    const int req = i / blocks, row0 = (blocks - 1 - i % blocks) * kTall, n = c.starts[req + 1] - c.starts[req];
    const int to = min(n, c.max_rows);
    const int ctx = max(0, min(c.seq_lens[req], c.max_blocks * c.cache.block_size));
    s_tokens[i] = row0 < to ? max(0, ctx - n + min(to, row0 + kTall)) : -1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
    int place = 0;
    for (int k = 0; k < pairs; ++k) place += s_tokens[k] > s_tokens[i] || (s_tokens[k] == s_tokens[i] && k < i);
    if (place == rank) s_pair = i;
  }
  __syncthreads();
  return s_pair;
}

template <typename T, int D, int kTiles>
__global__ void __launch_bounds__((kSoftWarp + 4 * kTiles) * 32, kTiles == 1 ? 2 : 1)
kv8_tile_kernel(const Kv8Call c, const Kv8Parts parts, const int blocks, const uint32_t blocks_magic, const int vec) {
  constexpr uint32_t kQSlab = kRows * 128, kSlab = kKeys * 128, kQBytes = D / 64 * kQSlab, kTileBytes = D / 64 * kSlab;
  constexpr uint32_t kCols = 256 * kTiles, kO = 128;   // tensor memory of a row tile: S (and P over it), then O
  extern __shared__ uint8_t smem_raw[];
  const uint32_t q_at = (smem_u32(smem_raw) + 1023) & ~1023u, k_at = q_at + kTiles * kQBytes, v_at = k_at + 2 * kTileBytes;
  __shared__ Aux<kTiles> aux;
  chain_wait();
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int splits = parts.splits, split = blockIdx.x % splits, head = blockIdx.x / splits % c.cache.heads;
  const int pair = longest_first<kTiles * kRows>(c, blocks, blockIdx.x / splits / c.cache.heads), req = pair / blocks;
  if (blockIdx.x == 0 && threadIdx.x == 0) parts.plan[kPlanStatus] = kStatusOk;
  const int start = c.starts[req], n_rows = c.starts[req + 1] - start, row0 = (blocks - 1 - pair % blocks) * (kTiles * kRows);
  const int rows_to = min(n_rows, c.max_rows);   // rows behind those are left as they are
  if (row0 >= rows_to) { chain_next(); return; }
  const int bs = c.cache.block_size, ctx = max(0, min(c.seq_lens[req], c.max_blocks * bs));
  const int first = ctx - n_rows + row0;                                 // own position of the CTA's first row
  const int rows_here = min(kTiles * kRows, rows_to - row0);
  const int end = first + rows_here;                                     // tokens that its last row attends to, if any
  const int all_tiles = max(0, (end + kKeys - 1) / kKeys), per = (all_tiles + splits - 1) / splits;
  const int tile0 = min(all_tiles, split * per), n_tiles = min(all_tiles, tile0 + per) - tile0;
  const int key0 = tile0 * kKeys;
  // warps without a row of the request leave the weights to chance: their rows of O are nobody's
  auto soft_warps = [&](int tile) { return min(4, max(0, rows_here - tile * kRows + 31) / 32); };
  if (threadIdx.x == 0) {
    mbar_init(&aux.q_full, 4 * kTiles);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&aux.k_full[i], kCopyWarps); mbar_init(&aux.v_full[i], kCopyWarps); mbar_init(&aux.k_empty[i], 1); mbar_init(&aux.v_empty[i], 1);
      for (int t = 0; t < kTiles; ++t) {
        mbar_init(&aux.s_full[t][i], 1); mbar_init(&aux.p_full[t][i], max(1, soft_warps(t))); mbar_init(&aux.o_done[t][i], 1);
      }
    }
    for (int i = 0; i < 4; ++i) mbar_init(&aux.scales_full[i], kCopyWarps);
    aux.abort_flag = 0;
    mbar_init_fence();
  }
  if (warp == 0) tmem_alloc(&aux.tmem_base, kCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  chain_next();
  const uint32_t tmem = aux.tmem_base;
  volatile int* abort_flag = &aux.abort_flag;
  int* status = parts.plan + kPlanStatus;
  auto wait = [&](uint64_t* bars, int tile) {
    return mbar_wait_warp(smem_u32(&bars[tile & 1]), (uint32_t)(tile >> 1) & 1u, abort_flag, status, kStatusTileWait, lane);
  };
  auto wait_two = [&](uint64_t* a, int i, uint64_t* b, int j) {   // both round trips at once
    const bool there = mbar_try_wait_addr(smem_u32(&a[i & 1]), (uint32_t)(i >> 1) & 1u) & mbar_try_wait_addr(smem_u32(&b[j & 1]), (uint32_t)(j >> 1) & 1u);
    return __all_sync(0xffffffffu, there) || (wait(a, i) && wait(b, j));
  };
  auto arrive = [&](uint64_t* bar) {   // what the warp has written to shared memory is the tensor cores'
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) mbar_arrive_addr(smem_u32(bar));
  };
  bool ok = true;
  if (warp >= 1 && warp < kSoftWarp) {
    // ---- codes to fp16: every warp its groups of 16 tokens (which never straddle a block) of a key tile ----
    constexpr int kPieces = D / 16, kAtOnce = 32 / kPieces, kLoads = 16 / kAtOnce;   // 16-byte pieces of a row, rows at once
    constexpr int kMine = kGroups / kCopyWarps;
    const int piece = lane % kPieces, r0 = lane / kPieces;
    const int32_t* table = c.tables + (int64_t)req * c.max_blocks;
    const int64_t row_bytes = (int64_t)c.cache.heads * D, column = (int64_t)head * D + piece * 16 + r0 * row_bytes;
    const uint32_t per_block = (uint32_t)bs / 16;
    const int odd = piece / 4 & 1;   // the second slab's pieces in the other order: 8 lanes, 8 different bank groups
    const int mine = warp - 1;
    struct Place { int64_t from; int block, rows; };   // rows that count; none: no block of the cache, or behind the last token
    auto block_of = [&](int g) {   // of the group's tokens; group / per_block by the high word of a product
      const uint32_t group = (uint32_t)key0 / 16 + g;
      return key0 + g * 16 < end ? table[blocks_magic ? __umulhi(group, blocks_magic) : group] : -1;
    };
    auto place = [&](int g, int block) {
      const uint32_t group = (uint32_t)key0 / 16 + g, at = blocks_magic ? __umulhi(group, blocks_magic) : group;
      Place p;
      const bool in = block >= 0 && block < c.cache.num_blocks;
      p.rows = in ? min(16, end - key0 - g * 16) : -1;
      p.block = in ? block : 0;   // something that can be read
      p.from = p.block * c.cache.block_stride + (int64_t)((group - at * per_block) * 16) * row_bytes + column;
      return p;
    };
    auto load = [&](uint4 (&codes)[kLoads], const uint8_t* cache, const Place& p) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) codes[i] = ld_ahead(cache + p.from + i * kAtOnce * row_bytes);
    };
    auto store = [&](uint32_t tile, const uint4 (&codes)[kLoads], int rows_from) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int row = rows_from + r0 + i * kAtOnce;
        const uint32_t base = tile + piece / 4 * kSlab + row * 128;
        const uint4 w = codes[i];
        const uint32_t half[2][2] = {{odd ? w.z : w.x, odd ? w.w : w.y}, {odd ? w.x : w.z, odd ? w.y : w.w}};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t x[4];
#pragma unroll
          for (int e = 0; e < 2; ++e) e4m3x4_to_f16x4(half[h][e], x[2 * e], x[2 * e + 1]);
          st_shared16(base + (((piece % 4 * 2 + (h ^ odd)) ^ (row & 7)) << 4), x);
        }
      }
    };
    // a tile's codes are on their way while the last one's are handed over; the table's entries one tile further ahead
    uint4 k[kMine][kLoads], v[kMine][kLoads];
    Place now[kMine];
    int next[kMine];
    float2 scale[kMine];
    auto load_scale = [&](const Place& p) {
      const int64_t at = p.block * c.cache.scale_stride + head;
      return make_float2(c.cache.key_scale[at], c.cache.value_scale[at]);
    };
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      now[i] = place(mine + i * kCopyWarps, n_tiles > 0 ? block_of(mine + i * kCopyWarps) : -1);
      load(k[i], c.cache.key, now[i]);
      scale[i] = load_scale(now[i]);
      load(v[i], c.cache.value, now[i]);
      next[i] = n_tiles > 1 ? block_of(kGroups + mine + i * kCopyWarps) : -1;
    }
    for (int j = 0; j < n_tiles; ++j) {
      const int i2 = j & 1;
      Place then[kMine];
      if (j > 1 && !wait(aux.k_empty, j - 2)) { ok = false; break; }
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int q = mine + i * kCopyWarps;
        if (lane == 0)   // a block outside the cache: the scores of its tokens are NaN (those behind the last one are masked)
          aux.scales[j & 3][q] = now[i].rows < 0 ? make_float2(__int_as_float(0x7fc00000), -INFINITY) : make_float2(scale[i].x, log2f(scale[i].y));
        store(k_at + i2 * kTileBytes, k[i], q * 16);
        then[i] = place((j + 1) * kGroups + q, next[i]);
        load(k[i], c.cache.key, then[i]);
        scale[i] = load_scale(then[i]);
        next[i] = j + 2 < n_tiles ? block_of((j + 2) * kGroups + q) : -1;
      }
      if (lane == 0) mbar_arrive_addr(smem_u32(&aux.scales_full[j & 3]));
      arrive(&aux.k_full[i2]);
      if (j > 1 && !wait(aux.v_empty, j - 2)) { ok = false; break; }
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int q = mine + i * kCopyWarps;
        if (now[i].rows < 16) {   // rows that do not count have no weight, but zero times whatever they hold might be NaN
#pragma unroll
          for (int e = 0; e < kLoads; ++e)
            if (r0 + e * kAtOnce >= now[i].rows) v[i][e] = make_uint4(0, 0, 0, 0);
        }
        store(v_at + i2 * kTileBytes, v[i], q * 16);
        load(v[i], c.cache.value, then[i]);
        now[i] = then[i];
      }
      arrive(&aux.v_full[i2]);
    }
  } else if (warp == 0) {
    // ---- products ----
    constexpr uint32_t s_idesc = mma_idesc(0, 128, kKeys, false);
    constexpr uint32_t o_idesc = mma_idesc(0, 128, D, false) | (1u << 16);   // B is MN-major
    // descriptors' low halves: an offset in shared memory adds its sixteenth
    const uint32_t q_lo = desc_lo(q_at, 16), k_lo = desc_lo(k_at, 16), v_lo = desc_lo(v_at, kSlab);
    const int used = kTiles == 2 && soft_warps(1) > 0 ? 2 : 1;   // a second row tile without rows has no products: nobody would wait for them
    auto scores = [&](int j) {   // S of key tile j
      if (elect_one()) {
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          if (t >= used) break;
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            tc_mma_cta(tmem + t * 256 + (j & 1) * kKeys, q_lo + (t * kQBytes + k / 4 * kQSlab + k % 4 * 32) / 16, desc_hi(1024, true),
                       k_lo + (j & 1) * (kTileBytes / 16) + (k / 4 * kSlab + k % 4 * 32) / 16, desc_hi(1024, true), s_idesc, k != 0);
          tc_commit_cta(smem_u32(&aux.s_full[t][j & 1]));
        }
        tc_commit_cta(smem_u32(&aux.k_empty[j & 1]));
      }
      __syncwarp();
    };
    auto values = [&](int t, int j) {
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k)
          mma_tmem_a(tmem + t * 256 + kO, tmem + t * 256 + (j & 1) * kKeys + k * 8, v_lo + (j & 1) * (kTileBytes / 16) + k * 128,
                     desc_hi(1024, true), o_idesc, j > 0 || k != 0);
        tc_commit_cta(smem_u32(&aux.o_done[t][(j & 1)]));
        if (t == used - 1) tc_commit_cta(smem_u32(&aux.v_empty[j & 1]));
      }
      __syncwarp();
    };
    if (n_tiles > 0) {
      ok = mbar_wait_warp(smem_u32(&aux.q_full), 0, abort_flag, status, kStatusTileWait, lane) && wait(aux.k_full, 0);
      tc_fence_after();
      if (ok) scores(0);
    }
    for (int j = 0; j < n_tiles && ok; ++j) {
      if (j + 1 < n_tiles) {   // S of the next key tile, into the buffer that held the weights of tile j - 1
        ok = j > 0 ? wait_two(aux.k_full, j + 1, aux.v_empty, j - 1) : wait(aux.k_full, 1);
        if (!ok) break;
        tc_fence_after();
        scores(j + 1);
      }
      ok = wait_two(aux.v_full, j, aux.p_full[0], j);
      if (!ok) break;
      tc_fence_after();
      values(0, j);
      if constexpr (kTiles == 2) {
        if (used < 2) continue;
        ok = wait(aux.p_full[1], j);
        if (!ok) break;
        tc_fence_after();
        values(1, j);
      }
    }
    // tensor memory and barriers are given up when every product has ended and its arrivals are there
    for (int j = max(0, n_tiles - 2); j < n_tiles && ok; ++j) {
      ok = wait(aux.k_empty, j) && wait(aux.v_empty, j);
      for (int t = 0; t < used && ok; ++t) ok = wait(aux.o_done[t], j);
    }
  } else {
    // ---- softmax: a thread per row; the warp's quarter of tensor memory is its number modulo 4 ----
    const int tile = (warp - kSoftWarp) / 4, quarter = warp & 3, row = tile * kRows + quarter * 32 + lane;
    const uint32_t lanes = tmem + tile * 256 + ((uint32_t)(quarter * 32) << 16), o_at = lanes + kO;
    const int64_t t = (int64_t)start + row0 + row;
    const bool mine = row < rows_here && t >= 0 && t < c.rows;
    const bool live = quarter < soft_warps(tile);
    float up = 1.f;   // what the row's scores are multiplied by for its query's fp16 form
    {
      const T* src = static_cast<const T*>(c.query) + (mine ? t : 0) * c.query_stride + (int64_t)head * D;
      uint4 q[D / 8];   // the whole row at once: one round trip
#pragma unroll
      for (int e = 0; e < D / 8; ++e) q[e] = make_uint4(0, 0, 0, 0);
      if (mine && vec) {
#pragma unroll
        for (int e = 0; e < D / 8; ++e) q[e] = ld_ahead(reinterpret_cast<const uint8_t*>(src + 8 * e));
      } else if (mine) {
#pragma unroll
        for (int e = 0; e < D / 8; ++e) {
          struct alignas(16) { T x[8]; } some;
#pragma unroll
          for (int i = 0; i < 8; ++i) some.x[i] = src[8 * e + i];
          q[e] = *reinterpret_cast<const uint4*>(&some);
        }
      }
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < D / 8; ++e) {
          float x[8];
          Vec16<T>::unpack(q[e], x);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (fabsf(x[i]) <= 3.402823466e38f) top = fmaxf(top, fabsf(x[i]));
        }
        // the largest element to 2^14 ... 2^15; factors within fp32's normal range
        const int p = min(120, 127 + 14 - (int)(__float_as_uint(top) >> 23));
        const float down = __uint_as_float((uint32_t)(127 + p) << 23);
        up = __uint_as_float((uint32_t)(127 - p) << 23);
#pragma unroll
        for (int e = 0; e < D / 8; ++e) {
          float x[8];
          Vec16<T>::unpack(q[e], x);
          q[e] = make_uint4(half2_bits(x[0] * down, x[1] * down), half2_bits(x[2] * down, x[3] * down),
                            half2_bits(x[4] * down, x[5] * down), half2_bits(x[6] * down, x[7] * down));
        }
      }
#pragma unroll
      for (int e = 0; e < D / 8; ++e)
        st_shared16(q_at + tile * kQBytes + e / 8 * kQSlab + (row % kRows) * 128 + (((e & 7) ^ (row & 7)) << 4),
                    reinterpret_cast<const uint32_t*>(&q[e]));
      arrive(&aux.q_full);
    }
    const float coef = parts.scale_log2 * up;
    float m = -INFINITY, l = 0.f, ref = -INFINITY;
    for (int j = 0; j < n_tiles && live; ++j) {
      const uint32_t s_at = lanes + (j & 1) * kKeys;
      const int seen = first + row - key0 - j * kKeys;   // the last token of the key tile that the row attends to
      const bool diagonal = key0 + j * kKeys + kKeys - 1 > first + tile * kRows;
      const float2* scales = aux.scales[j & 3];
      const uint32_t s_bar = smem_u32(&aux.s_full[tile][(j & 1)]), s_parity = (uint32_t)(j >> 1) & 1u;
      const uint32_t f_bar = smem_u32(&aux.scales_full[j & 3]), f_parity = (uint32_t)(j >> 2) & 1u;
      const bool there = mbar_try_wait_addr(f_bar, f_parity) & mbar_try_wait_addr(s_bar, s_parity);   // both round trips at once
      if (!__all_sync(0xffffffffu, there) && !(mbar_wait_warp(f_bar, f_parity, abort_flag, status, kStatusTileWait, lane) &&
                                               mbar_wait_warp(s_bar, s_parity, abort_flag, status, kStatusTileWait, lane))) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t v[kKeys];
      tmem_ld32(s_at, v);
      tmem_ld32(s_at + 32, v + 32);
      float by[kGroups], lv[kGroups], m_new = m, r_new = -INFINITY;
#pragma unroll
      for (int b = 0; b < kGroups; ++b) {
        by[b] = coef * scales[b].x;
        lv[b] = scales[b].y;
      }
      tmem_ld_wait32(v);
      tmem_ld_wait32(v + 32);
      if (diagonal) {
        // -infinity times a factor that is 0 or NaN would be NaN: such a factor goes into the scores
#pragma unroll
        for (int b = 0; b < kGroups; ++b) {
          const bool plain = by[b] > 0.f;
          const uint32_t fill = by[b] == 0.f ? 0u : 0x7fc00000u;
          if (!plain) by[b] = 1.f;
#pragma unroll
          for (int i = 16 * b; i < 16 * b + 16; ++i) v[i] = i > seen ? 0xff800000u : plain ? v[i] : fill;
        }
      }
#pragma unroll
      for (int b = 0; b < kGroups; ++b) {
        float tops[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 16 * b; i < 16 * b + 16; i += 2)
          tops[i / 2 & 1] = max3(tops[i / 2 & 1], __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
        const float top = fmaxf(tops[0], tops[1]) * by[b];   // NaN counts as none
        m_new = fmaxf(m_new, top);
        r_new = fmaxf(r_new, top + lv[b]);
      }
      if (j == 0) {
        ref = r_new;
      } else {
        const bool move = r_new > ref && !(r_new - ref <= kSlack);
        if (__any_sync(0xffffffffu, move)) {
          if (!wait(aux.o_done[tile], j - 1)) { ok = false; break; }   // O is as the last tile left it
          tc_fence_after();
          const float down = move && ref != -INFINITY ? ex2(ref - r_new) : 1.f;
          if (move) ref = r_new;
#pragma unroll 1
          for (int d = 0; d < D; d += 16) {
            uint32_t o[16];
            tmem_ld16(o_at + d, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * down);
            tmem_st16(o_at + d, o);
          }
        }
      }
      const float shift = m_new == -INFINITY ? 0.f : m_new, base = shift - (ref == -INFINITY ? 0.f : ref) + kUp;
      l *= m == -INFINITY ? 0.f : ex2(m - shift);
      m = m_new;
      // the weights as they meet V, 2^(x + off): their sums go back to the scores' own reference block by block.  A block whose off is
      // below -60 has no weight in fp16 either way
#pragma unroll
      for (int b = 0; b < kGroups; ++b) {
        const float at = base + lv[b], off = at < -60.f ? -60.f : at, from = off - shift;
        float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int i = 16 * b; i < 16 * b + 16; i += 2) {
          float2 x = fma2(make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), by[b], from);
          x.x = ex2(x.x);
          x.y = ex2(x.y);
          sums[i / 2 & 1] = add2(sums[i / 2 & 1], x);
          v[i / 2] = half2_bits(x.x, x.y);
        }
        sums[0] = add2(sums[0], sums[1]);
        l = fmaf(sums[0].x + sums[0].y, ex2(-off), l);
        if (b & 1) tmem_st16(s_at + 8 * (b - 1), v + 8 * (b - 1));
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_addr(smem_u32(&aux.p_full[tile][(j & 1)]));
    }
    ok = ok && (n_tiles == 0 || !live || wait(aux.o_done[tile], n_tiles - 1));
    tc_fence_after();
    const float bad = __int_as_float(0x7fc00000);
    // O is relative to 2^(ref - kUp), the sum and the parts to 2^m; in two steps, with the least scales the factor is 2^-133, below the
    // normal range
    const float root = ref == -INFINITY ? 0.f : ex2(0.5f * (ref - kUp - (m == -INFINITY ? 0.f : m)));
    float by = root;
    const bool none = first + row < 0;    // a row before the first token
    const int64_t unit = (t * c.cache.heads + head) * splits + split;
    if (splits == 1) by /= l;             // nothing but scores of -infinity: NaN
    if (!ok) by = bad;
    if (none) by = 0.f;
    T* out = static_cast<T*>(c.out) + t * c.out_stride + (int64_t)head * D;
#pragma unroll
    for (int d = 0; d < D; d += 16) {
      uint32_t o[16];
      if (n_tiles > 0 && live) {
        tmem_ld16(o_at + d, o);
        tmem_ld_wait();
      }
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = none || n_tiles == 0 || !live ? 0.f : __uint_as_float(o[i]) * root * by;
      if (mine && splits > 1) {
        float* dst = parts.acc + unit * D + d;
#pragma unroll
        for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(dst + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
      } else if (mine && vec) {
        struct alignas(16) Eight { T x[8]; };
#pragma unroll
        for (int i = 0; i < 16; i += 8) {
          Eight e;
#pragma unroll
          for (int k = 0; k < 8; ++k) e.x[k] = Elem<T>::from_float(x[i + k]);
          *reinterpret_cast<Eight*>(out + d + i) = e;
        }
      } else if (mine) {
#pragma unroll
        for (int i = 0; i < 16; ++i) out[d + i] = Elem<T>::from_float(x[i]);
      }
    }
    if (splits > 1 && mine) parts.ml[unit] = make_float2(ok ? m : 0.f, ok ? l : bad);
  }
  if (!ok) {   // products still in flight get a bounded time to end
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) { }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) { tc_fence_after(); tmem_free(tmem, kCols); }
}

template <typename T, int D, int kTiles>
int launch(const Kv8Call& c, const Kv8Parts& parts, cudaStream_t stream) {
  static bool done[64] = {false};
  auto kernel = kv8_tile_kernel<T, D, kTiles>;
  constexpr size_t smem = tile_smem<D, kTiles>();
  int dev = 0;
  APS_CUDA(cudaGetDevice(&dev));
  APS_REQUIRE(dev >= 0 && dev < 64, APS_ERR_CUDA, "device index %d out of range", dev);
  if (!done[dev]) {
    APS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    APS_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
    done[dev] = true;
  }
  const int vec = aligned_to(c.query, 16) && aligned_to(c.out, 16) && c.query_stride % 8 == 0 && c.out_stride % 8 == 0;
  const int blocks = (c.max_rows + kTiles * kRows - 1) / (kTiles * kRows);
  const int64_t grid = (int64_t)c.batch * blocks * c.cache.heads * parts.splits;
  APS_REQUIRE(grid < (int64_t(1) << 31), APS_ERR_SHAPE, "kv8_attention: too many rows");
  return launch_chained("kv8_tile_kernel", kernel, (unsigned)grid, (kSoftWarp + 4 * kTiles) * 32, smem, stream, c, parts, blocks,
                        kv8_blocks_magic(c.cache.block_size), vec);
}

// Row tiles per CTA: two save a tenth where they are filled (six chunks of 500 rows 185 us, with one 205); where the requests' average
// would leave more of them empty (43 requests of 109 rows, some more than 128: 342 us, with one 322) one.
int tiles_of(const Kv8Call& c) {
  const int64_t rows = (c.rows + c.batch - 1) / c.batch, one = (rows + kRows - 1) / kRows * kRows, two = (rows + 2 * kRows - 1) / (2 * kRows) * (2 * kRows);
  return c.max_rows > kRows && two * 10 <= one * 11 ? 2 : 1;
}

template <typename T>
int launch_typed(const Kv8Call& c, const Kv8Parts& parts, cudaStream_t stream) {
  const bool two = tiles_of(c) == 2;
  if (c.cache.head_size == 128) return two ? launch<T, 128, 2>(c, parts, stream) : launch<T, 128, 1>(c, parts, stream);
  return two ? launch<T, 64, 2>(c, parts, stream) : launch<T, 64, 1>(c, parts, stream);
}

}  // namespace

bool kv8_tiles_take(const Kv8Call& c) {
  // the maximum is taken of the raw scores: a scale that is not positive would need their minimum
  return c.starts != nullptr && c.max_rows > 1 && (c.dtype == APS_F16 || c.dtype == APS_BF16) &&
         (c.cache.head_size == 64 || c.cache.head_size == 128) && c.cache.num_blocks > 0 && c.scale >= 1.17549435e-38f && c.scale < 1.70141183e38f;
}

// Parts that the tokens of a tile of rows are cut into: as many as the GPU takes at a time (a few CTAs more would run alone in the end:
// 503 rows of 9 heads at 4879 tokens, 162 CTAs 54 us, 144 33), eight key tiles each at least.
int kv8_tile_splits(const Kv8Call& c, int tiles) {
  const int64_t key_tiles = ((int64_t)c.max_blocks * c.cache.block_size + 63) / 64, rows = (int64_t)tiles * kRows;
  const int64_t row_tiles = (c.rows + rows - 1) / rows, units = (row_tiles > c.batch ? row_tiles : c.batch) * c.cache.heads;
  int64_t n = (int64_t)sm_count() * (tiles == 1 ? 2 : 1) / units;
  if (n > (key_tiles + 7) / 8) n = (key_tiles + 7) / 8;
  return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
}
int kv8_tile_splits(const Kv8Call& c) { return kv8_tile_splits(c, tiles_of(c)); }

int launch_kv8_tiles(const Kv8Call& c, const Kv8Parts& parts, cudaStream_t stream) {
  return c.dtype == APS_BF16 ? launch_typed<__nv_bfloat16>(c, parts, stream) : launch_typed<__half>(c, parts, stream);
}

}  // namespace aps
