// Matrix products of the gated feed-forward block on the tensor cores (tcgen05, TMEM, TMA).
//
// One persistent CTA per SM (or a pair of CTAs on two SMs that share a 256-row tile): warp 16
// copies operand tiles of 64 of K into a ring in shared memory (TMA, 128-byte swizzle), warp 17
// issues the MMAs into one of two TMEM accumulators, and warps 0-15 turn the other accumulator
// into results, 16 columns of 32 rows at a time. Operands may lie along K or across it in memory: the tile copies and the MMA
// descriptors follow, nothing is transposed in a pass of its own.
#include "gemm_tc.cuh"

#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "tcgen05.cuh"

namespace fhb {
namespace {

constexpr int kKBlock = 64;                      // K of one ring slot: 128 bytes of bf16
constexpr int kRows = 128;                       // result rows of one CTA
constexpr int kMaxColumns = 256;                 // result columns of a tile
constexpr int kEpilogueWarps = 16;
constexpr int kGroup = 16;                       // columns that a thread works on together
constexpr int kThreads = 32 * (kEpilogueWarps + 2);
constexpr int kMaxSlots = 16;
constexpr int kRingBytes = 216 * 1024;
constexpr int kPlanes = 3;                       // of an FP32 operand
constexpr int kMaxOperands = 5;  // of a block's products
constexpr int kATileBytes = kRows * kKBlock * 2;  // 16 KB: of 128 rows, all of which an MMA reads

// Of a launch of Jobs products. A launch of one has its own kernels: constants at places that are
// known when they are compiled (looked up by product, they cost large products 8%, small ones more).
template <int Jobs>
struct Maps {
  CUtensorMap a[Jobs][2], b[Jobs][2];
};

// One product of a launch.
struct Job {
  int64_t m, n;               // result rows and columns (gate: n hidden features, 2 n columns)
  int tiles_m, tiles_n, groups, parts;
  int k_blocks, part_blocks;  // of K, and of each part of K
  int sum_terms;
  int a_k_major, b_k_major;
  // rows of one A copy: fewer than 128 where m is small (the MMAs then read what follows as the
  // other rows, whose results are not used)
  int a_rows;
  uint32_t idesc;
  uint32_t first_item;
  // results: out + bias, or FP32 sums of each part of K
  void* out[2];
  int64_t out_stride;
  int out_wide;               // 32-byte stores are aligned
  const void* bias[2];
  float* partial;
  int64_t partial_stride;
};
struct Common {
  int jobs;
  uint32_t items;
  int columns;                // columns of a tile (both halves of a gate tile)
  int slots, slot_blocks;     // of the ring; blocks of K in a slot
  uint32_t slot_bytes;
  bf16* gated[2];
  int64_t gated_stride, gated_plane;
  TcFactors factors;
  int activation;
  float* row_sums;            // [32 rows][dg, du][row_sums_stride]: their column sums, or null
  int64_t row_sums_stride;
  unsigned int* status;
};
template <int Jobs>
struct Args : Common {
  Job job[Jobs];
};

// ---- PTX pieces that the other kernels' header does not have ----

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t in_cta(uint32_t smem, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem), "r"(rank));
  return r;
}
__device__ __forceinline__ void arrive_remote(uint32_t bar) {
  // relaxed: what it orders are TMEM reads, by the tcgen05 fence before it; a release would wait
  // for the thread's stores to memory (3,000 cycles a tile)
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

template <int Cg>
__device__ __forceinline__ void copy_tile(uint32_t dst, const CUtensorMap* map, int x, int y, int z,
                                          uint32_t bar) {
  if (Cg == 2)
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        ".cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}

// Shared-memory matrix descriptor of a tile in 128-byte swizzle. K-major: rows of 128 bytes
// (64 of K), groups of 8 rows 1024 bytes apart (`lbo` unused). MN-major: blocks of 64 rows or
// columns, each 64 of K by 128 bytes; `lbo` between blocks, 1024 bytes between 8 of K.
__device__ __forceinline__ uint64_t tile_descriptor(uint32_t smem, uint32_t lbo) {
  return static_cast<uint64_t>((smem >> 4) & 0x3FFFu) |
         (static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16) |
         (static_cast<uint64_t>(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// The four MMAs (K = 16 each) of one ring slot, issued by one elected lane of a converged warp.
template <int Cg>
__device__ __forceinline__ void mma_slot(uint32_t d, uint64_t a, uint64_t b, uint32_t a_step,
                                         uint32_t b_step, uint32_t idesc, uint32_t accumulate) {
#define FHB_MMA_SLOT(GROUP)                                                             \
  asm volatile(                                                                         \
      "{\n\t.reg .pred e, p, t;\n\t.reg .b64 a1, a2, a3, b1, b2, b3, sa, sb;\n\t"       \
      "setp.ne.b32 p, %6, 0;\n\tsetp.eq.b32 t, %6, %6;\n\t"                             \
      "cvt.u64.u32 sa, %3;\n\tcvt.u64.u32 sb, %4;\n\t"                                  \
      "add.u64 a1, %1, sa;\n\tadd.u64 a2, a1, sa;\n\tadd.u64 a3, a2, sa;\n\t"           \
      "add.u64 b1, %2, sb;\n\tadd.u64 b2, b1, sb;\n\tadd.u64 b3, b2, sb;\n\t"           \
      "elect.sync _|e, 0xffffffff;\n\t"                                                 \
      "@e tcgen05.mma.cta_group::" GROUP ".kind::f16 [%0], %1, %2, %5, p;\n\t"          \
      "@e tcgen05.mma.cta_group::" GROUP ".kind::f16 [%0], a1, b1, %5, t;\n\t"          \
      "@e tcgen05.mma.cta_group::" GROUP ".kind::f16 [%0], a2, b2, %5, t;\n\t"          \
      "@e tcgen05.mma.cta_group::" GROUP ".kind::f16 [%0], a3, b3, %5, t;\n\t}" ::"r"(d), \
      "l"(a), "l"(b), "r"(a_step), "r"(b_step), "r"(idesc), "r"(accumulate)             \
      : "memory")
  if (Cg == 2)
    FHB_MMA_SLOT("2");
  else
    FHB_MMA_SLOT("1");
#undef FHB_MMA_SLOT
}

// Arrives on `bar` (in both CTAs of a pair) when the MMAs issued so far are done.
template <int Cg>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if (Cg == 2)
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster"
        ".multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(smem_u32(bar)),
        "h"(static_cast<uint16_t>(3))
        : "memory");
  else
    tc::commit_warp(bar);
}

template <int Cg>
__device__ __forceinline__ void allocate_tmem(uint32_t* dst) {
  if (Cg == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(dst)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tc::tmem_alloc(dst, 512);
    tc::tmem_relinquish();
  }
}
template <int Cg>
__device__ __forceinline__ void free_tmem(uint32_t tmem) {
  if (Cg == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  else
    tc::tmem_dealloc(tmem, 512);
}

// 32 bytes in one access, 32-byte aligned: a whole memory sector per thread.
__device__ __forceinline__ void store32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void load32(const void* p, uint32_t* v) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]),
                 "=r"(v[6]), "=r"(v[7])
               : "l"(p)
               : "memory");
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// x and y as sums of three bf16 each, w[i] holding the i-th pieces of both: each piece is the
// remainder rounded to 8 significant bits, so every difference is exact, the second piece is at most
// 2^-8 of x and the third 2^-17, with either sign. Their sum is x (from 2^-110 up; below it, x to the
// 2^-133 at which bf16 ends). What would round up to infinity is cut instead; an infinity is all in
// the first piece.
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&w)[3]) {
  constexpr float kRoundsUp = 0x1.FFp127f;
  const auto low = [](uint32_t v) { return __uint_as_float(v << 16); };
  const auto high = [](uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); };
  w[0] = pack_bf16(x, y);
  float rest_x = x - low(w[0]), rest_y = y - high(w[0]);
  if (!(fabsf(x) < kRoundsUp && fabsf(y) < kRoundsUp)) {
    const bool real_x = fabsf(x) < INFINITY, real_y = fabsf(y) < INFINITY;
    w[0] = pack_bf16(real_x ? high(__float_as_uint(x)) : x, real_y ? high(__float_as_uint(y)) : y);
    rest_x = real_x ? x - low(w[0]) : 0.0f;
    rest_y = real_y ? y - high(w[0]) : 0.0f;
  }
  w[1] = pack_bf16(rest_x, rest_y);
  w[2] = pack_bf16(rest_x - low(w[1]), rest_y - high(w[1]));
}

// Where a lane's row lies among its neighbours': rows of lanes 2i and 2i + 1 are written together.
struct RowPair {
  bool odd, even_row, odd_row;  // this lane's place; which of the two rows exist
};
// 64 bytes of each lane's row at `p` (rows `stride` bytes apart from lane to lane), in two pieces:
// the lanes of a pair exchange one, so that an access has 64 bytes of a row (5.8 TB/s where 32
// bytes a row reach 4.3). For whole warps.
__device__ __forceinline__ void store64(void* p, int64_t stride, const RowPair& rows,
                                        const uint32_t (&first)[8], const uint32_t (&second)[8]) {
  uint32_t got[8], w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) got[i] = __shfl_xor_sync(0xffffffffu, rows.odd ? first[i] : second[i], 1);
  char* const at = static_cast<char*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = rows.odd ? got[i] : first[i];
  if (rows.even_row) store32(rows.odd ? at - stride + 32 : at, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = rows.odd ? second[i] : got[i];
  if (rows.odd_row) store32(rows.odd ? at + 32 : at + stride, w);
}
// 16 FP32 values of each lane's row.
__device__ __forceinline__ void store64(float* p, int64_t stride, const RowPair& rows, const float (&v)[kGroup]) {
  uint32_t a[8], b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = __float_as_uint(v[i]), b[i] = __float_as_uint(v[8 + i]);
  store64(static_cast<void*>(p), stride * 4, rows, a, b);
}
__device__ __forceinline__ void pack_group(const float (&v)[kGroup], uint32_t (&w)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
}

// 16 values of a row in operand form (bf16, or three planes), 32-byte aligned.
template <typename T>
__device__ __forceinline__ void store_operand(bf16* p, int64_t plane, const float (&v)[kGroup]) {
  uint32_t w[8];
  if (sizeof(T) == 2) {
    pack_group(v, w);
    store32(p, w);
  } else {
    uint32_t w1[8], w2[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t pieces[3];
      split_pair(v[2 * i], v[2 * i + 1], pieces);
      w[i] = pieces[0];
      w1[i] = pieces[1];
      w2[i] = pieces[2];
    }
    store32(p, w);
    store32(p + plane, w1);
    store32(p + 2 * plane, w2);
  }
}

// 16 results of a row from column n0 on, those below n.
template <typename T>
__device__ __forceinline__ void store_results(T* row, int64_t n0, int64_t n, bool wide,
                                              const float (&v)[kGroup]) {
  T* p = row + n0;
  if (wide && n0 + kGroup <= n) {
    uint32_t w[16];
    if (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
      store32(p, w);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[i]);
      store32(p, w);
      store32(p + 8, w + 8);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kGroup; ++i)
    if (n0 + i < n) p[i] = from_float<T>(v[i]);
}

// Adds bias[n0 + i], the same for all lanes: in 16-byte loads where all 16 exist.
template <typename T>
__device__ __forceinline__ void add_bias(const void* bias, int64_t n0, int64_t n, float (&v)[kGroup]) {
  if (bias == nullptr) return;
  const T* p = static_cast<const T*>(bias) + n0;
  if (n0 + kGroup <= n && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    constexpr int kEach = 16 / sizeof(T);
    uint4 w[kGroup / kEach];
#pragma unroll
    for (int i = 0; i < kGroup / kEach; ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
#pragma unroll
    for (int i = 0; i < kGroup / kEach; ++i) {
      const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (sizeof(T) == 4) {
          v[4 * i + j] += __uint_as_float(u[j]);
        } else {
          v[8 * i + 2 * j] += __uint_as_float(u[j] << 16);
          v[8 * i + 2 * j + 1] += __uint_as_float(u[j] & 0xFFFF0000u);
        }
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kGroup; ++i)
    if (n0 + i < n) v[i] += to_float(p[i]);
}

// The power of 2 that brings a group's largest magnitude into [2^14, 2^15), the top of f16's
// range (values down to 2^-28 of the largest keep f16's 11 bits), from its FP32 exponent e,
// kept where the power and its inverse are normal FP32 numbers.
__device__ __forceinline__ float group_scale(float largest, uint32_t& e) {
  e = min(max(__float_as_uint(largest) >> 23, 15u), 254u);
  return __uint_as_float((268u - e) << 23);
}
__device__ __forceinline__ float group_unscale(uint32_t e) {
  return __uint_as_float((e - 14u) << 23);
}

// The factors of a group of 16, both kinds, into their places (see TcFactors). For whole warps.
__device__ __forceinline__ uint32_t pack_factors(const float (&v)[kGroup], uint32_t (&w)[8]) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < kGroup; ++i) top = fmaxf(top, fabsf(v[i]));
  if (!(top < INFINITY)) {  // an infinity stays one at any scale: the others set it
    top = 0.0f;
#pragma unroll
    for (int i = 0; i < kGroup; ++i) top = fmaxf(top, fabsf(v[i]) < INFINITY ? fabsf(v[i]) : 0.0f);
  }
  uint32_t e;
  const float scale = group_scale(top, e);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i] * scale, v[2 * i + 1] * scale);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return e;
}
template <typename T>
__device__ __forceinline__ void store_factors(const TcFactors& f, int64_t place, bool own, const RowPair& rows,
                                              const float (&f1)[kGroup], const float (&f2)[kGroup]) {
  const int64_t row_values = f.groups * 2 * kFactorGroup;  // from one token to the next
  if constexpr (sizeof(T) == 2) {
    uint32_t a[8], b[8];
    const uint32_t e1 = pack_factors(f1, a), e2 = pack_factors(f2, b);
    store64(static_cast<__half*>(f.values) + place * kFactorGroup, row_values * 2, rows, a, b);
    if (own) *reinterpret_cast<uint16_t*>(f.exponents + place) = static_cast<uint16_t>(e1 | e2 << 8);
  } else {
    float* p = static_cast<float*>(f.values) + place * kFactorGroup;
    store64(p, row_values, rows, f1);
    store64(p + kFactorGroup, row_values, rows, f2);
  }
}
// The factors of one kind of a group, as they lie in memory.
template <typename T>
struct FactorWords {
  uint32_t w[4 * sizeof(T)];
  uint32_t exponent;
};
template <typename T>
__device__ __forceinline__ void load_factors(const TcFactors& f, int64_t place, FactorWords<T>& x) {
  const char* p = static_cast<const char*>(f.values) + place * (kFactorGroup * sizeof(T));
  load32(p, x.w);
  if (sizeof(T) == 4) load32(p + 32, x.w + 8);
  if (sizeof(T) == 2) x.exponent = f.exponents[place];
}
// out[i] = v[i] times factor i
template <typename T>
__device__ __forceinline__ void times_factors(const FactorWords<T>& x, const float (&v)[kGroup], float (&out)[kGroup]) {
  if constexpr (sizeof(T) == 2) {
    const float unscale = group_unscale(x.exponent);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x.w[i]));
      out[2 * i] = v[2 * i] * (f.x * unscale);
      out[2 * i + 1] = v[2 * i + 1] * (f.y * unscale);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kGroup; ++i) out[i] = v[i] * __uint_as_float(x.w[i]);
  }
}

// Column sums over the 16 lanes of a lane's parity: lane l gets column l / 2's, by halving the
// columns and doubling the rows, in a fixed order.
__device__ __forceinline__ float sum_rows(const float (&v)[kGroup], int lane) {
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float keep = lane & 16 ? v[i + 8] : v[i], give = lane & 16 ? v[i] : v[i + 8];
    s[i] = keep + __shfl_xor_sync(0xffffffffu, give, 16);
  }
#pragma unroll
  for (int half = 4; half >= 1; half /= 2)
#pragma unroll
    for (int i = 0; i < half; ++i) {
      const bool upper = lane & (2 * half);
      const float keep = upper ? s[i + half] : s[i], give = upper ? s[i] : s[i + half];
      s[i] = keep + __shfl_xor_sync(0xffffffffu, give, 2 * half);
    }
  return s[0];
}

template <int Jobs>
__device__ __forceinline__ const Job& job_of(const Args<Jobs>& p, int job) {
  return p.job[Jobs == 1 ? 0 : job];
}

// One item of work: a tile of one group's result of a product, and one part of K.
struct Item {
  int job, group, part, first_block, blocks;
  int64_t m0, n0;  // first row of the tile (of the pair), first column (gate: feature)
};
// (32-bit divisions: there are fewer than 2^31 items, and 64-bit ones took 3,000 cycles an item)
template <int Cg, bool Gate, int Jobs>
__device__ __forceinline__ Item item_at(const Args<Jobs>& p, uint32_t index) {
  Item it;
  it.job = 0;
  if constexpr (Jobs > 1)
    while (it.job + 1 < p.jobs && index >= p.job[it.job + 1].first_item) ++it.job;
  const Job& q = job_of(p, it.job);
  if constexpr (Jobs > 1) index -= q.first_item;
  const uint32_t tiles = static_cast<uint32_t>(q.tiles_m) * static_cast<uint32_t>(q.tiles_n);
  const uint32_t rest = index / tiles;
  uint32_t tile = index - rest * tiles;
  it.group = static_cast<int>(rest / q.parts);
  it.part = static_cast<int>(rest) - it.group * q.parts;
  // bands of 8 tile rows, column by column: the tiles in flight share their operands in L2
  const uint32_t band_tiles = 8u * static_cast<uint32_t>(q.tiles_n), band = tile / band_tiles;
  const uint32_t rows = min(8u, static_cast<uint32_t>(q.tiles_m) - 8u * band);
  tile -= band * band_tiles;
  const uint32_t column = tile / rows;
  it.m0 = static_cast<int64_t>(8u * band + (tile - column * rows)) * (kRows * Cg);
  it.n0 = static_cast<int64_t>(column) * (Gate ? p.columns / 2 : p.columns);
  it.first_block = it.part * q.part_blocks;
  it.blocks = min(q.part_blocks, q.k_blocks - it.first_block);
  return it;
}

// FP32 blocks. A slot holds the three planes of 64 of K of both operands, for six of their nine
// products (the others come to at most 2^-24 of a product, of either sign): the large one has an
// accumulator of its own and the five small ones share another, kSmallColumns on. The tensor core
// cuts each sum to FP32 instead of rounding it, an error that grows with the number of additions and
// has a sign: the small products do not add to it that way, and K is summed in chunks of
// kChunkBlocks slots per term, the chunks in registers, rounded.
constexpr int kChunkBlocks = 2;
constexpr int kSmallColumns = 128;
template <typename T>
__device__ __forceinline__ int chunk_count(int blocks) {
  return sizeof(T) == 4 ? (blocks + kChunkBlocks - 1) / kChunkBlocks : 1;
}

template <int Cg, TcEpilogue E, typename T, int Jobs>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_tc_kernel(const __grid_constant__ Maps<Jobs> maps, const __grid_constant__ Args<Jobs> p) {
  constexpr bool kGateTile = E == TcEpilogue::kGate;
  constexpr bool kChunked = sizeof(T) == 4;
  constexpr int kCopies = kChunked ? kPlanes : 1;  // planes that come with one copy
  extern __shared__ unsigned char raw[];
  __shared__ uint64_t full[kMaxSlots], empty[kMaxSlots], sum_full[2], sum_empty[2];
  __shared__ uint32_t tmem_at;
  const uint32_t ring = (smem_u32(raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = Cg == 2 ? cluster_rank() : 0;
  const int b_rows = p.columns / Cg;  // rows of this CTA's B tile
  const uint32_t b_tile_bytes = static_cast<uint32_t>(b_rows) * kKBlock * 2;
  const uint32_t slot_bytes = p.slot_bytes;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.slots; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sum_full[i], 1);
      mbar_init(&sum_empty[i], kEpilogueWarps * Cg);
    }
    fence_barrier_init();
  }
  if (warp == kEpilogueWarps) allocate_tmem<Cg>(&tmem_at);
  tc::fence_before_sync();
  __syncthreads();
  if (Cg == 2) cluster_sync();
  tc::fence_after_sync();
  const uint32_t tmem = tmem_at;
  // launched as a dependent of the kernel before it: the set-up above runs beside that one's
  // end, and nothing of its results, nor of what it still reads, is touched before this wait
  allow_dependents();
  wait_for_prerequisites();

  const uint32_t items = p.items;
  const uint32_t first = blockIdx.x / Cg, stride = gridDim.x / Cg;

  if (warp == kEpilogueWarps) {
    // ---- copies ----
    if (lane == 0) {
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      int64_t issued = 0;
      const uint32_t first_bar = Cg == 2 ? in_cta(smem_u32(&full[0]), 0) : smem_u32(&full[0]);
      for (uint32_t index = first; ok && index < items; index += stride) {
        const Item it = item_at<Cg, kGateTile, Jobs>(p, index);
        const Job& q = job_of(p, it.job);
        const uint32_t a_tile_bytes = static_cast<uint32_t>(q.a_rows) * kKBlock * 2;
        const uint32_t block_bytes = kCopies * (a_tile_bytes + b_tile_bytes);  // of one block of K
        const bool a_k_major = q.a_k_major != 0, b_k_major = q.b_k_major != 0;
        const int chunks = chunk_count<T>(it.blocks);
        const int a0 = static_cast<int>(it.m0 + rank * kRows);
        const int b0 = static_cast<int>(it.n0) + (kGateTile ? 0 : static_cast<int>(rank) * b_rows);
        for (int c = 0; ok && c < chunks; ++c) {
          const int low = it.first_block + (kChunked ? c * kChunkBlocks : 0);
          const int high = kChunked ? min(low + kChunkBlocks, it.first_block + it.blocks)
                                    : it.first_block + it.blocks;
          for (int t = 0; ok && t < q.sum_terms; ++t) {
            const CUtensorMap* am = &maps.a[Jobs == 1 ? 0 : it.job][q.groups == 2 ? it.group : t];
            const CUtensorMap* bm = &maps.b[Jobs == 1 ? 0 : it.job][kGateTile && Cg == 2 ? static_cast<int>(rank) : t];
            for (int kb = low; kb < high; kb += p.slot_blocks) {
              if (!mbar_wait_bounded(&empty[slot], phase ^ 1, p.status, FHB_STATUS_MMA_TIMEOUT)) {
                ok = false;
                break;
              }
              const int blocks = min(p.slot_blocks, high - kb);
              if (rank == 0) mbar_arrive_expect_tx(&full[slot], Cg * block_bytes * blocks);
              const uint32_t bar = first_bar + slot * 8;
              for (int j = 0; j < blocks; ++j) {
                const uint32_t at = ring + slot * slot_bytes + j * block_bytes;
                const uint32_t bt = at + kCopies * a_tile_bytes;
                const int k0 = (kb + j) * kKBlock;
                if (a_k_major) {
                  copy_tile<Cg>(at, am, k0, a0, 0, bar);
                } else {
                  copy_tile<Cg>(at, am, a0, k0, 0, bar);
                  copy_tile<Cg>(at + kCopies * 8192, am, a0 + 64, k0, 0, bar);
                }
                if (kGateTile && Cg == 1) {
                  // half of the columns from each weight; FP32: plane by plane, so that the
                  // halves of a plane are neighbours
                  for (int z = 0; z < kCopies; ++z) {
                    copy_tile<Cg>(bt + z * b_tile_bytes, &maps.b[0][0], k0, b0, z, bar);
                    copy_tile<Cg>(bt + z * b_tile_bytes + b_tile_bytes / 2, &maps.b[0][1], k0, b0, z, bar);
                  }
                } else if (b_k_major) {
                  copy_tile<Cg>(bt, bm, k0, b0, 0, bar);
                } else {
                  for (int i = 0; i < b_rows; i += 64)
                    copy_tile<Cg>(bt + i * kCopies * 128, bm, b0 + i, k0, 0, bar);
                }
              }
              ++issued;
              if (++slot == p.slots) {
                slot = 0;
                phase ^= 1;
              }
            }
          }
        }
      }
      // the last copies have landed before this CTA's memory is given up, also where a wait gave up
      // (a pair's barriers are in CTA 0, and its CTAs leave together)
      if (rank == 0)
        for (int s = 0; s < p.slots && issued > 0; ++s, --issued) {
          slot = slot == 0 ? p.slots - 1 : slot - 1;
          if (slot == p.slots - 1) phase ^= 1;
          mbar_wait_bounded(&full[slot], phase, p.status, FHB_STATUS_MMA_TIMEOUT);
        }
    }
    __syncwarp();
  } else if (warp == kEpilogueWarps + 1) {
    // ---- MMAs (a pair's are issued by its first CTA) ----
    if (rank == 0) {
      int slot = 0;
      uint32_t phase = 0;
      int64_t sums = 0;
      bool ok = true, begun = false;
      // (operand across K: bytes from one block of 64 rows to the next)
      const uint64_t a_desc = tile_descriptor(0, kCopies * 8192), b_desc = a_desc;
      for (uint32_t index = first; ok && index < items; index += stride) {
        const Item it = item_at<Cg, kGateTile, Jobs>(p, index);
        const Job& q = job_of(p, it.job);
        const uint32_t a_step = q.a_k_major ? 2 : 128, b_step = q.b_k_major ? 2 : 128;  // 16 of K
        const uint32_t a_tile_bytes = static_cast<uint32_t>(q.a_rows) * kKBlock * 2;
        const uint32_t block_bytes = kCopies * (a_tile_bytes + b_tile_bytes);
        // bytes from plane to plane
        const uint32_t a_plane = q.a_k_major ? a_tile_bytes : 8192;
        const uint32_t b_plane = q.b_k_major ? b_tile_bytes : 8192;
        const uint32_t idesc = q.idesc;
        const int sum_terms = q.sum_terms;
        const int chunks = chunk_count<T>(it.blocks);
        for (int c = 0; ok && c < chunks; ++c, ++sums) {
          const int low = kChunked ? c * kChunkBlocks : 0;
          const int blocks = kChunked ? min(kChunkBlocks, it.blocks - low) : it.blocks;
          const int buffer = static_cast<int>(sums & 1);
          ok = mbar_wait_bounded(&sum_empty[buffer], static_cast<uint32_t>((sums >> 1) & 1) ^ 1,
                                 p.status, FHB_STATUS_MMA_TIMEOUT);
          if (!ok) break;
          tc::fence_after_sync();
          const uint32_t d = tmem + buffer * kMaxColumns;
          uint32_t accumulate = 0;
          for (int t = 0; ok && t < sum_terms; ++t)
            for (int kb = 0; kb < blocks; kb += p.slot_blocks) {
              ok = mbar_wait_bounded(&full[slot], phase, p.status, FHB_STATUS_MMA_TIMEOUT);
              if (!ok) break;
              tc::fence_after_sync();
              const uint32_t at = ring + slot * slot_bytes;
              if constexpr (kChunked) {
                const uint32_t bt = at + kCopies * a_tile_bytes;
                const uint64_t a0 = a_desc | (at >> 4), b0 = b_desc | (bt >> 4);
                const uint64_t a1 = a0 + (a_plane >> 4), b1 = b0 + (b_plane >> 4);
                const uint64_t a2 = a1 + (a_plane >> 4), b2 = b1 + (b_plane >> 4);
                const uint32_t small = d + kSmallColumns;
                mma_slot<Cg>(small, a2, b0, a_step, b_step, idesc, accumulate);
                mma_slot<Cg>(d, a0, b0, a_step, b_step, idesc, accumulate);
                mma_slot<Cg>(small, a0, b2, a_step, b_step, idesc, 1);
                mma_slot<Cg>(small, a1, b1, a_step, b_step, idesc, 1);
                mma_slot<Cg>(small, a1, b0, a_step, b_step, idesc, 1);
                mma_slot<Cg>(small, a0, b1, a_step, b_step, idesc, 1);
                accumulate = 1;
              } else {
                const int here = min(p.slot_blocks, blocks - kb);
                uint64_t a0 = a_desc | (at >> 4), b0 = b_desc | ((at + a_tile_bytes) >> 4);
                for (int j = 0; j < here; ++j) {
                  mma_slot<Cg>(d, a0, b0, a_step, b_step, idesc, accumulate);
                  accumulate = 1;
                  a0 += block_bytes >> 4;
                  b0 += block_bytes >> 4;
                }
              }
              commit<Cg>(&empty[slot]);
              begun = true;
              if (++slot == p.slots) {
                slot = 0;
                phase ^= 1;
              }
            }
          if (ok) commit<Cg>(&sum_full[buffer]);
        }
      }
      // the last MMAs are done before their accumulators and operands are given up, likewise
      if (begun) {
        slot = slot == 0 ? p.slots - 1 : slot - 1;
        if (slot == p.slots - 1) phase ^= 1;
        mbar_wait_bounded(&empty[slot], phase, p.status, FHB_STATUS_MMA_TIMEOUT);
      }
    }
    __syncwarp();
  } else {
    // ---- results: each warp has 32 rows; four warps share the columns ----
    const int quadrant = warp % 4, quarter = warp / 4, pairs = p.columns / 32;
    // a warp's pairs of 16 columns are neighbours
    const int each = (pairs + 3) / 4, first_pair = quarter * each, end_pair = min(pairs, first_pair + each);
    const uint32_t release = Cg == 2 ? in_cta(smem_u32(&sum_empty[0]), 0) : smem_u32(&sum_empty[0]);
    int64_t sums = 0;
    bool ok = true;
    for (uint32_t index = first; ok && index < items; index += stride) {
      const Item it = item_at<Cg, kGateTile, Jobs>(p, index);
      const Job& q = job_of(p, it.job);
      const int chunks = chunk_count<T>(it.blocks);
      const int64_t row = it.m0 + rank * kRows + quadrant * 32 + lane;
      const bool odd = (lane & 1) != 0, own = row < q.m;
      const RowPair rows{odd, row - odd < q.m, row + !odd < q.m};
      const auto release_sums = [&](int buffer) {
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if (Cg == 2) arrive_remote(release + buffer * 8);
          else mbar_arrive(&sum_empty[buffer]);
        }
      };
      // waits for the sums of a chunk of K; the warps agree, since what follows is for whole warps
      const auto wait_sums = [&](int buffer) {
        ok = mbar_wait_bounded(&sum_full[buffer], static_cast<uint32_t>((sums >> 1) & 1), p.status,
                               FHB_STATUS_MMA_TIMEOUT);
        ok = __all_sync(0xffffffffu, ok);
        tc::fence_after_sync();
        return ok;
      };
      const uint32_t lanes = static_cast<uint32_t>(quadrant * 32) << 16;
      // 16 columns of the sums over K: FP32 blocks add both accumulators and their chunks
      const auto add_columns = [&](uint32_t at, bool first, float (&v)[kGroup]) {
        __syncwarp();
        if constexpr (kChunked) {
          float more[kGroup];
          tc::ld_x16(at + kSmallColumns, more);
          if (first) {
            tc::ld_x16(at, v);
            tc::wait_ld();
#pragma unroll
            for (int i = 0; i < kGroup; ++i) v[i] += more[i];
          } else {
            float large[kGroup];
            tc::ld_x16(at, large);
            tc::wait_ld();
#pragma unroll
            for (int i = 0; i < kGroup; ++i) v[i] += large[i] + more[i];
          }
        } else {
          tc::ld_x16(at, v);
          tc::wait_ld();
        }
      };

      if constexpr (E == TcEpilogue::kGateGrad) {
        // Two groups of 16 columns at a time. The lanes of a pair exchange one, so that a lane has
        // one group of both rows and an access 64 bytes of a row (FP32, 65,536 x 64 -> 256: 117 ->
        // 104 us). A row's factors are on their way while the sums or the row before are worked on;
        // both rows' at once spill registers (16,384 x 2,048 -> 5,632, bf16: 374 us against 356).
        FactorWords<T> f1, f2;
        const auto prefetch = [&](int pair, int which_row) {
          const int64_t n0 = it.n0 + 32 * pair + 16 * odd, at_row = row - odd + which_row;
          if (at_row >= q.m || n0 >= q.n) return;
          const int64_t place = (at_row * p.factors.groups + n0 / kFactorGroup) * 2;
          load_factors<T>(p.factors, place, f1);
          load_factors<T>(p.factors, place + 1, f2);
        };
        const auto finish = [&](int pair, float (&v0)[kGroup], float (&v1)[kGroup]) {
          if (it.n0 + 32 * pair >= q.n) return;
          __syncwarp();
#pragma unroll
          for (int i = 0; i < kGroup; ++i) {
            const float got = __shfl_xor_sync(0xffffffffu, odd ? v0[i] : v1[i], 1);
            v0[i] = odd ? got : v0[i];
            v1[i] = odd ? v1[i] : got;
          }
          const int64_t n0 = it.n0 + 32 * pair + 16 * odd, first_row = it.m0 + rank * kRows + quadrant * 32;
          float sum[2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int64_t at_row = row - odd + r;
            const bool live = at_row < q.m && n0 < q.n;
            if (r == 1) prefetch(pair, 1);
#pragma unroll
            for (int which = 0; which < 2; ++which) {  // dg = dh f2, then du = dh f1
              float d[kGroup];
              times_factors<T>(which == 0 ? f2 : f1, r == 0 ? v0 : v1, d);
              if (live) store_operand<T>(p.gated[which] + at_row * p.gated_stride + n0, p.gated_plane, d);
              if (p.row_sums == nullptr) continue;
              if (!live) {
#pragma unroll
                for (int i = 0; i < kGroup; ++i) d[i] = 0.0f;
              }
              __syncwarp();
              const float s = sum_rows(d, lane);
              sum[which] = r == 0 ? s : sum[which] + s;
              if (r == 1 && first_row < q.m && n0 < q.n)
                p.row_sums[(first_row / 32 * 2 + which) * p.row_sums_stride + n0 + lane / 2] = sum[which];
            }
          }
        };
        if (first_pair < end_pair) prefetch(first_pair, 0);
        if constexpr (kChunked) {
          float v0[kGroup], v1[kGroup];  // at most 128 columns: a pair a warp
          for (int c = 0; c < chunks; ++c, ++sums) {
            const int buffer = static_cast<int>(sums & 1);
            if (!wait_sums(buffer)) break;
            if (first_pair < end_pair) {
              const uint32_t from = tmem + buffer * kMaxColumns + lanes + 32 * first_pair;
              add_columns(from, c == 0, v0);
              add_columns(from + 16, c == 0, v1);
            }
            release_sums(buffer);
          }
          if (ok && first_pair < end_pair) finish(first_pair, v0, v1);
        } else {
          const int buffer = static_cast<int>(sums & 1);
          if (!wait_sums(buffer)) break;
          ++sums;
          const uint32_t from = tmem + buffer * kMaxColumns + lanes;
          for (int pair = first_pair; pair < end_pair; ++pair) {
            float v0[kGroup], v1[kGroup];
            add_columns(from + 32 * pair, true, v0);
            add_columns(from + 32 * pair + 16, true, v1);
            if (pair + 1 == end_pair) release_sums(buffer);
            finish(pair, v0, v1);
            if (pair + 1 < end_pair) prefetch(pair + 1, 0);
          }
          if (first_pair >= end_pair) release_sums(buffer);
        }
      } else {
        // two groups of 16 columns at a time: a gate tile's g and u, else neighbours
        uint32_t held[8];  // bf16: h of the first of two neighbours, stored with the second's
        bool holds = false;
        const auto finish = [&](int pair, float (&v0)[kGroup], float (&v1)[kGroup]) {
          if constexpr (kGateTile) {
            const int64_t n0 = it.n0 + 16 * pair;
            if (n0 >= q.n) return;
            add_bias<T>(q.bias[0], n0, q.n, v0);
            add_bias<T>(q.bias[1], n0, q.n, v1);
            float h[kGroup];
            const auto gate = [&](auto tanh) {
#pragma unroll
              for (int i = 0; i < kGroup; ++i) {
                float a, slope;
                block_activation<decltype(tanh)::value>(v0[i], a, slope);
                h[i] = a * v1[i];
                v0[i] = a;
                v1[i] *= slope;
              }
            };
            if (p.activation == FHB_ACTIVATION_TANH) gate(std::true_type{});
            else gate(std::false_type{});
            __syncwarp();
            bf16* const at = p.gated[0] + row * p.gated_stride + n0;
            if constexpr (sizeof(T) == 2) {
              if (holds) {
                uint32_t w[8];
                pack_group(h, w);
                store64(at - kGroup, p.gated_stride * 2, rows, held, w);
                holds = false;
              } else if (pair + 1 < end_pair && n0 + kGroup < q.n) {
                pack_group(h, held);
                holds = true;
              } else if (own) {
                store_operand<T>(at, p.gated_plane, h);
              }
            } else if (own) {
              store_operand<T>(at, p.gated_plane, h);
            }
            if (p.factors.values != nullptr) {
              const int64_t place = (row * p.factors.groups + n0 / kFactorGroup) * 2;
              __syncwarp();
              store_factors<T>(p.factors, place, own, rows, v0, v1);
            }
          } else {
            const int64_t n0 = it.n0 + 32 * pair;
            if (n0 >= q.n) return;
            __syncwarp();
            if (q.partial != nullptr) {
              float* out = q.partial +
                           ((static_cast<int64_t>(it.group) * q.parts + it.part) * q.m + row) * q.partial_stride + n0;
              store64(out, q.partial_stride, rows, v0);
              store64(out + kGroup, q.partial_stride, rows, v1);
              return;
            }
            add_bias<T>(q.bias[0], n0, q.n, v0);
            if (n0 + kGroup < q.n) add_bias<T>(q.bias[0], n0 + kGroup, q.n, v1);
            T* const out = static_cast<T*>(q.out[it.group]) + row * q.out_stride;
            if (q.out_wide && n0 + 2 * kGroup <= q.n) {
              __syncwarp();
              if constexpr (sizeof(T) == 2) {
                uint32_t a[8], b[8];
                pack_group(v0, a);
                pack_group(v1, b);
                store64(out + n0, q.out_stride * 2, rows, a, b);
              } else {
                store64(out + n0, q.out_stride, rows, v0);
                store64(out + n0 + kGroup, q.out_stride, rows, v1);
              }
            } else if (own) {
              store_results<T>(out, n0, q.n, q.out_wide != 0, v0);
              store_results<T>(out, n0 + kGroup, q.n, q.out_wide != 0, v1);
            }
          }
        };
        float acc0[kGroup], acc1[kGroup];
        for (int c = 0; c < chunks; ++c, ++sums) {
          const int buffer = static_cast<int>(sums & 1);
          if (!wait_sums(buffer)) break;
          const uint32_t from = tmem + buffer * kMaxColumns + lanes;
          // FP32 blocks have at most 128 columns: a pair a warp, kept over the chunks
          for (int pair = first_pair; pair < end_pair; ++pair) {
            const uint32_t c0 = from + (kGateTile ? 16 * pair : 32 * pair);
            const uint32_t c1 = kGateTile ? from + p.columns / 2 + 16 * pair : c0 + 16;
            add_columns(c0, !kChunked || c == 0, acc0);
            add_columns(c1, !kChunked || c == 0, acc1);
            if (pair + 1 == end_pair) release_sums(buffer);
            if (!kChunked || c + 1 == chunks) finish(pair, acc0, acc1);
          }
          // a tile of 64 columns leaves half of the warps idle
          if (first_pair >= end_pair) release_sums(buffer);
        }
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (Cg == 2) cluster_sync();
  if (warp == kEpilogueWarps) free_tmem<Cg>(tmem);
}

// i / d of non-negative numbers, in 32 bits where they fit.
__device__ __forceinline__ int64_t quotient(int64_t i, int64_t d) {
  return (i | d) >> 32 == 0 ? static_cast<uint32_t>(i) / static_cast<uint32_t>(d) : i / d;
}

// out[m][n] = the sum of the parts in order + bias[n]; one group of a product per blockIdx.y.
struct Parts {
  const float* partial;
  int64_t part_values, stride, m, n, out_stride;
  int parts;
  const void* bias;
  void* out;
};
struct PartsList {
  Parts of[2 * kTcMaxProducts];
};
template <typename T>
__global__ void __launch_bounds__(256) add_parts_kernel(const __grid_constant__ PartsList list) {
  allow_dependents();
  wait_for_prerequisites();
  const Parts& p = list.of[blockIdx.y];
  const int64_t quads = p.stride / 4, step = p.part_values / 4;
  const T* const bias = static_cast<const T*>(p.bias);
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < p.m * quads; i += gridDim.x * 256ll) {
    const int64_t row = quotient(i, quads), c = (i - row * quads) * 4;
    const float4* src = reinterpret_cast<const float4*>(p.partial + row * p.stride + c);
    float4 s = src[0];
    int k = 1;
    for (; k + 4 <= p.parts; k += 4) {  // four parts in flight
      float4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = src[(k + j) * step];
#pragma unroll
      for (int j = 0; j < 4; ++j) s = make_float4(s.x + v[j].x, s.y + v[j].y, s.z + v[j].z, s.w + v[j].w);
    }
    for (; k < p.parts; ++k) {
      const float4 v = src[k * step];
      s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
    }
    const float v[4] = {s.x, s.y, s.z, s.w};
    T* const out = static_cast<T*>(p.out) + row * p.out_stride + c;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < p.n) out[j] = from_float<T>(v[j] + (bias != nullptr ? to_float(bias[c + j]) : 0.0f));
  }
}

// Rows of `cols` values into rows of `stride` bf16 (a multiple of 8, the rest zero): copies, or
// the three planes of FP32 values. One matrix per blockIdx.y.
struct PackJob {
  const void* in;
  bf16* out;
  int64_t rows, cols, in_stride, stride, plane;
};
struct PackJobs {
  PackJob job[kMaxOperands];
};
template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ PackJobs jobs) {
  allow_dependents();
  const PackJob& j = jobs.job[blockIdx.y];
  const int64_t pieces = j.stride / 8;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < j.rows * pieces; i += gridDim.x * 256ll) {
    const int64_t row = quotient(i, pieces), c = (i - row * pieces) * 8;
    const T* src = static_cast<const T*>(j.in) + row * j.in_stride + c;
    float v[8];
    if (sizeof(T) == 4 && c + 8 <= j.cols && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
      const float4 x = reinterpret_cast<const float4*>(src)[0], y = reinterpret_cast<const float4*>(src)[1];
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = c + k < j.cols ? to_float(src[k]) : 0.0f;
    }
    bf16* dst = j.out + row * j.stride + c;
    uint32_t w[3][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (sizeof(T) == 2) {
        w[0][k] = pack_bf16(v[2 * k], v[2 * k + 1]);
      } else {
        uint32_t pieces[3];
        split_pair(v[2 * k], v[2 * k + 1], pieces);
#pragma unroll
        for (int q = 0; q < 3; ++q) w[q][k] = pieces[q];
      }
    }
#pragma unroll
    for (int q = 0; q < (sizeof(T) == 2 ? 1 : 3); ++q)
      *reinterpret_cast<uint4*>(dst + q * j.plane) = make_uint4(w[q][0], w[q][1], w[q][2], w[q][3]);
  }
}

int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
int64_t blocks_of(int64_t x, int64_t size) { return (x + size - 1) / size; }

// ---- the plan of a launch: tile, pairing, each product's parts of K ----
struct JobPlan {
  int a_rows, parts, part_blocks, k_blocks, tiles_m, tiles_n;
  int64_t partial_stride;
};
struct Plan {
  int cg, columns, slots, slot_blocks, slot_bytes, grid;
  bool cut_rows;  // some A tile has fewer than 128 rows
  int64_t items;
  double cycles;  // the estimate
  JobPlan job[kTcMaxProducts];
};
// Bytes of the ring that one block of K takes.
int block_bytes_of(bool wide, int cg, int columns, int a_rows) {
  return (wide ? kPlanes : 1) * (a_rows + columns / cg) * kKBlock * 2;
}

// Chooses by an estimate of the launch's cycles. A block of K costs its MMAs (4 x columns / 2
// cycles a product of planes, the same in a pair with half the B tile each) or the copies of its
// bytes (about 64 a cycle), whichever is longer; an item costs about 2,000 cycles more (its
// first copies, its last results), and a second launch that adds the parts about 3,000 and its
// bytes. So a few tokens get tiles as narrow as still fill one round of the SMs (48 x 2048 x 5632
// bf16, first product: 14.1 us with 118 tiles of 96 columns, 14.6 with 88 of 128, 19.7 with 176
// of 64), and products that share a launch are cut so that no item is long against the launch.
Plan plan_of(const TcProduct* products, int count, const DeviceInfo& dev) {
  const bool wide = products[0].dtype == FHB_DTYPE_F32, gate = products[0].epilogue == TcEpilogue::kGate;
  const bool parted = products[0].epilogue == TcEpilogue::kStore;
  Plan best{};
  double least = 0.0;
  for (int cg = 1; cg <= 2; ++cg)
    for (const int columns : {64, 96, 128, 192, 256}) {
      bool fits = columns <= (wide ? kSmallColumns : kMaxColumns) && (cg == 1 || columns >= 128);
      for (int i = 0; i < count; ++i) {
        // an operand across K comes in blocks of 64
        if (!products[i].b_k_major && columns / cg % 64 != 0) fits = false;
        if (cg == 2 && products[i].m <= kRows) fits = false;
      }
      if (!fits) continue;
      const int64_t units = dev.sms / cg;
      Plan plan{};
      plan.cg = cg;
      plan.columns = columns;
      double block[kTcMaxProducts], whole = 0.0;
      int64_t tiles[kTcMaxProducts];
      for (int i = 0; i < count; ++i) {
        const TcProduct& p = products[i];
        JobPlan& j = plan.job[i];
        j.a_rows = p.a_k_major ? static_cast<int>(std::min<int64_t>(kRows, round_up(p.m, 8))) : kRows;
        j.k_blocks = static_cast<int>(blocks_of(p.k, kKBlock));
        j.tiles_m = static_cast<int>(blocks_of(p.m, kRows * cg));
        j.tiles_n = static_cast<int>(blocks_of(gate ? 2 * p.n : p.n, columns));
        j.partial_stride = round_up(p.n, 32);
        tiles[i] = static_cast<int64_t>(j.tiles_m) * j.tiles_n * p.groups;
        block[i] = p.sum_terms * std::max(2.0 * columns * (wide ? 6 : 1),
                                          block_bytes_of(wide, cg, columns, j.a_rows) / 64.0);
        whole += static_cast<double>(tiles[i]) * (2000.0 + j.k_blocks * block[i]) / static_cast<double>(units);
      }
      for (int choice = 1; choice <= (parted ? 6 : 1); ++choice) {
        double cycles = 0.0, longest = 0.0, added = 0.0;
        plan.items = 0;
        for (int i = 0; i < count; ++i) {
          const TcProduct& p = products[i];
          JobPlan& j = plan.job[i];
          int64_t wanted;
          if (count == 1)  // one to four parts, or as many as fill one or two rounds of the SMs
            wanted = choice <= 4 ? choice : units * (choice - 4) / tiles[0];
          else  // items of at most the whole, a half, ... a fifth of it; or no parts
            wanted = choice == 6 ? 1 : static_cast<int64_t>(j.k_blocks * block[i] * choice / whole) + 1;
          wanted = std::min<int64_t>(std::max<int64_t>(wanted, 1), 128);
          j.part_blocks = static_cast<int>(blocks_of(j.k_blocks, wanted));
          j.parts = static_cast<int>(blocks_of(j.k_blocks, j.part_blocks));
          const double item = 2000.0 + j.part_blocks * block[i];
          const int64_t items = tiles[i] * j.parts;
          plan.items += items;
          cycles += count == 1 ? static_cast<double>(blocks_of(items, units)) * item
                               : static_cast<double>(items) * item / static_cast<double>(units);
          longest = std::max(longest, item);
          if (j.parts > 1)
            added += 8.0 * static_cast<double>(p.m) * j.partial_stride * p.groups * j.parts / (64.0 * dev.sms);
        }
        if (count > 1) cycles += 0.5 * longest;
        if (added > 0.0) cycles += 3000.0 + added;
        if (least == 0.0 || cycles < least) {
          least = cycles;
          best = plan;
          best.cycles = cycles;
        }
      }
    }
  int block_bytes = 0, part_blocks = 0;
  for (int i = 0; i < count; ++i) {
    const JobPlan& j = best.job[i];
    block_bytes = std::max(block_bytes, block_bytes_of(wide, best.cg, best.columns, j.a_rows));
    part_blocks = std::max(part_blocks, j.part_blocks);
    best.cut_rows = best.cut_rows || j.a_rows < kRows;
  }
  const int room = kRingBytes - (best.cut_rows ? kATileBytes : 0);  // an MMA reads past the last rows
  // blocks of K a slot: two halve the waits between MMAs, where at least three slots remain; four
  // in narrow tiles, whose time is that of reading the weights: DRAM then gives 512 bytes of a
  // row together (48 x 2048 x 5632 bf16, 64 columns: 31, 23 and 20 us with 1, 2 and 4)
  best.slot_blocks = 1;
  for (const int blocks : {2, 4})
    if (!wide && part_blocks >= blocks && (blocks == 2 || best.columns < 128) && room / (blocks * block_bytes) >= 3)
      best.slot_blocks = blocks;
  best.slot_bytes = best.slot_blocks * block_bytes;
  best.slots = std::min(kMaxSlots, room / best.slot_bytes);
  return best;
}

// ---- TMA tile maps ----
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// The driver's encoder, looked up with the first product: null where the driver has none.
EncodeTiled encoder() {
  static const EncodeTiled found = [] {
    void* entry = nullptr;
    cudaDriverEntryPointQueryResult result;
    const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &entry, 12000,
                                                           cudaEnableDefault, &result);
    return e == cudaSuccess && result == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiled>(entry)
                                                                     : nullptr;
  }();
  return found;
}

// Tiles of 64 columns (128 bytes, swizzled) by `box_rows` rows of `box_planes` planes.
bool tile_map(const TcMatrix& x, int box_rows, int box_planes, CUtensorMap* out) {
  const cuuint64_t size[3] = {static_cast<cuuint64_t>(x.cols), static_cast<cuuint64_t>(x.rows),
                              static_cast<cuuint64_t>(x.planes)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(x.stride) * 2,
                                 static_cast<cuuint64_t>(x.planes > 1 ? x.plane : x.stride) * 2};
  const cuuint32_t box[3] = {kKBlock, static_cast<cuuint32_t>(box_rows),
                             static_cast<cuuint32_t>(box_planes)}, step[3] = {1, 1, 1};
  const EncodeTiled encode_tiled = encoder();
  if (encode_tiled == nullptr) return false;
  const auto encode = [&] {
    return encode_tiled(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<bf16*>(x.p), size, strides,
                    box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  if (encode()) return true;
  // the driver call needs a context on this thread, which the runtime makes current only with
  // the thread's first call that needs one (autograd's threads may not have made any)
  int device = 0;
  return cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess && encode();
}

size_t smem_bytes(const Plan& plan) {
  return static_cast<size_t>(plan.slots) * plan.slot_bytes + (plan.cut_rows ? kATileBytes : 0) + 1024;
}

// Lets a kernel have the ring's shared memory, with its first launch on a device: callers of the
// library's other operators do not wait for these kernels to load.
template <int Cg, TcEpilogue E, typename T, int Jobs>
cudaError_t allow_ring() {
  static std::atomic<uint64_t> allowed{0};  // a bit a device
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const uint64_t bit = uint64_t{1} << (device % 64);
  if ((allowed.load(std::memory_order_acquire) & bit) != 0) return cudaSuccess;
  e = cudaFuncSetAttribute(gemm_tc_kernel<Cg, E, T, Jobs>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           kRingBytes + 1024);
  if (e == cudaSuccess) allowed.fetch_or(bit, std::memory_order_release);
  return e;
}

template <int Cg, TcEpilogue E, typename T, int Jobs>
cudaError_t launch(const Maps<Jobs>& maps, const Args<Jobs>& args, const Plan& plan, bool dependent,
                   cudaStream_t stream) {
  const cudaError_t e = allow_ring<Cg, E, T, Jobs>();
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[2];
  int attrs = 0;
  if (Cg == 2) {
    attr[attrs].id = cudaLaunchAttributeClusterDimension;
    attr[attrs].val.clusterDim.x = Cg;
    attr[attrs].val.clusterDim.y = attr[attrs].val.clusterDim.z = 1;
    ++attrs;
  }
  if (dependent) {
    attr[attrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[attrs].val.programmaticStreamSerializationAllowed = 1;
    ++attrs;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(plan.grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem_bytes(plan);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = attrs;
  return cudaLaunchKernelEx(&cfg, gemm_tc_kernel<Cg, E, T, Jobs>, maps, args);
}

template <TcEpilogue E, int Jobs>
cudaError_t launch_kind(bool wide, const Maps<Jobs>& maps, const Args<Jobs>& args, const Plan& plan,
                        bool dependent, cudaStream_t stream) {
  if (wide)
    return plan.cg == 2 ? launch<2, E, float>(maps, args, plan, dependent, stream)
                        : launch<1, E, float>(maps, args, plan, dependent, stream);
  return plan.cg == 2 ? launch<2, E, bf16>(maps, args, plan, dependent, stream)
                      : launch<1, E, bf16>(maps, args, plan, dependent, stream);
}

// Short products go into one launch (see gemm_tc.cuh).
bool shares_launch(const Plan& plan) { return plan.cycles < 60000.0; }  // about 35 us

size_t parts_bytes(const TcProduct* products, int count, const Plan& plan) {
  size_t bytes = 0;
  for (int i = 0; i < count; ++i)
    if (plan.job[i].parts > 1)
      bytes += static_cast<size_t>(plan.job[i].parts) * products[i].groups * products[i].m *
               plan.job[i].partial_stride * 4;
  return bytes;
}

cudaError_t launch_planned(const TcProduct* products, int count, Plan plan, void* workspace,
                           bool dependent, const DeviceInfo& dev, cudaStream_t stream) {
  const TcProduct& p = products[0];
  const bool wide = p.dtype == FHB_DTYPE_F32, gate = p.epilogue == TcEpilogue::kGate;
  const int planes = wide ? kPlanes : 1;
  // items are counted in 32 bits, with room for a last stride beyond them
  if (plan.items > 0x70000000) return cudaErrorInvalidValue;
  Args<kTcMaxProducts> args{};
  Maps<kTcMaxProducts> maps{};
  PartsList parts{};
  int parted = 0;
  int64_t most = 0;
  float* partial = static_cast<float*>(workspace);
  args.columns = plan.columns;
  args.slots = plan.slots;
  args.slot_blocks = plan.slot_blocks;
  args.slot_bytes = static_cast<uint32_t>(plan.slot_bytes);
  uint32_t items = 0;
  for (int i = 0; i < count; ++i) {
    TcProduct x = products[i];
    const JobPlan& j = plan.job[i];
    // results that nobody wants: the plan is that of all of them, so that the others' sums are
    // made from the same parts either way
    if (p.epilogue == TcEpilogue::kStore) {
      if (x.groups == 2 && x.out[0] == nullptr) x.out[0] = x.out[1], x.a[0] = x.a[1], x.out[1] = nullptr;
      if (x.groups == 2 && x.out[1] == nullptr) x.groups = 1;
      if (x.out[0] == nullptr) continue;
    }
    const int at = args.jobs++;
    Job& q = args.job[at];
    q.m = x.m;
    q.n = x.n;
    q.tiles_m = j.tiles_m;
    q.tiles_n = j.tiles_n;
    q.groups = x.groups;
    q.parts = j.parts;
    q.k_blocks = j.k_blocks;
    q.part_blocks = j.part_blocks;
    q.sum_terms = x.sum_terms;
    q.a_k_major = x.a_k_major;
    q.b_k_major = x.b_k_major;
    q.a_rows = j.a_rows;
    q.idesc = (1u << 4) | (1u << 7) | (1u << 10) | (x.a_k_major ? 0u : tc::kIdescAMnMajor) |
              (x.b_k_major ? 0u : tc::kIdescBMnMajor) | (static_cast<uint32_t>(plan.columns) >> 3 << 17) |
              (static_cast<uint32_t>(kRows * plan.cg) >> 4 << 24);  // bf16 in, FP32 sums
    q.first_item = items;
    items += static_cast<uint32_t>(j.tiles_m) * j.tiles_n * x.groups * j.parts;
    q.out_stride = x.out_stride;
    const int64_t out_bytes = x.out_stride * static_cast<int64_t>(dtype_bytes(x.dtype));
    q.out_wide = out_bytes % 32 == 0 && reinterpret_cast<uintptr_t>(x.out[0]) % 32 == 0 &&
                 reinterpret_cast<uintptr_t>(x.out[1]) % 32 == 0;
    q.partial_stride = j.partial_stride;
    const int64_t values = x.m * j.partial_stride;
    for (int g = 0; g < 2; ++g) {
      q.out[g] = x.out[g];
      q.bias[g] = x.bias[g];
      if (j.parts == 1 || g >= x.groups) continue;
      if (g == 0) q.partial = partial;
      parts.of[parted++] = {partial, values, j.partial_stride, x.m, x.n, x.out_stride, j.parts, x.bias[0], x.out[g]};
      partial += j.parts * values;
      most = std::max(most, values);
    }
    const int a_box = x.a_k_major ? j.a_rows : kKBlock;
    const int b_box = !x.b_k_major ? kKBlock : gate ? plan.columns / 2 : plan.columns / plan.cg;
    for (int t = 0; t < 2; ++t) {
      if (x.a[t].p != nullptr && !tile_map(x.a[t], a_box, planes, &maps.a[at][t])) return cudaErrorInvalidValue;
      if (x.b[t].p != nullptr && !tile_map(x.b[t], b_box, gate && plan.cg == 1 ? 1 : planes, &maps.b[at][t]))
        return cudaErrorInvalidValue;
    }
  }
  if (items == 0) return cudaSuccess;
  args.items = items;
  plan.grid = static_cast<int>(std::min<int64_t>(items, dev.sms / plan.cg)) * plan.cg;
  for (int i = 0; i < 2; ++i) args.gated[i] = const_cast<bf16*>(p.gated[i].p);
  args.gated_stride = p.gated[0].stride;
  args.gated_plane = p.gated[0].plane;
  args.factors = p.factors;
  args.activation = p.activation;
  args.row_sums = p.row_sums;
  args.row_sums_stride = p.row_sums_stride;
  args.status = dev.status;
  cudaError_t e;
  if (args.jobs == 1) {
    Args<1> one{};
    static_cast<Common&>(one) = args;
    one.job[0] = args.job[0];
    Maps<1> of_one;
    for (int t = 0; t < 2; ++t) of_one.a[0][t] = maps.a[0][t], of_one.b[0][t] = maps.b[0][t];
    if (gate) return launch_kind<TcEpilogue::kGate>(wide, of_one, one, plan, dependent, stream);
    if (p.epilogue == TcEpilogue::kGateGrad)
      return launch_kind<TcEpilogue::kGateGrad>(wide, of_one, one, plan, dependent, stream);
    e = launch_kind<TcEpilogue::kStore>(wide, of_one, one, plan, dependent, stream);
  } else {
    e = launch_kind<TcEpilogue::kStore>(wide, maps, args, plan, dependent, stream);
  }
  if (e != cudaSuccess || parted == 0) return e;
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(blocks_of(most / 4, 256), 8ll * dev.sms)), parted);
  return launch_dependent(wide ? add_parts_kernel<float> : add_parts_kernel<bf16>, grid, dim3(256), 0, stream, parts);
}

}  // namespace

size_t gemm_tc_workspace_bytes(const TcProduct* products, int count, const DeviceInfo& dev) {
  const Plan plan = plan_of(products, count, dev);
  if (count == 1 || shares_launch(plan)) return parts_bytes(products, count, plan);
  size_t most = 0;
  for (int i = 0; i < count; ++i) most = std::max(most, gemm_tc_workspace_bytes(products + i, 1, dev));
  return most;
}

cudaError_t launch_gemm_tc(const TcProduct* products, int count, void* workspace, bool dependent,
                           const DeviceInfo& dev, cudaStream_t stream) {
  const Plan plan = plan_of(products, count, dev);
  if (count == 1 || shares_launch(plan))
    return launch_planned(products, count, plan, workspace, dependent, dev, stream);
  for (int i = 0; i < count; ++i) {
    const cudaError_t e = launch_planned(products + i, 1, plan_of(products + i, 1, dev), workspace,
                                         dependent || i > 0, dev, stream);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

namespace {
bool copies_by_tile(const void* p, int64_t stride, int dtype) {
  return dtype == FHB_DTYPE_BF16 && reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0;
}
}  // namespace

size_t tc_result_bytes(int64_t rows, int64_t cols, int dtype) {
  return static_cast<size_t>(rows) * round_up(cols, 32) * 2 * (dtype == FHB_DTYPE_F32 ? 3 : 1);
}

TcMatrix tc_result(void* room, int64_t rows, int64_t cols, int dtype) {
  const int64_t stride = round_up(cols, 32);
  return {static_cast<const bf16*>(room), rows, cols, stride, rows * stride, dtype == FHB_DTYPE_F32 ? 3 : 1};
}

size_t tc_operand_bytes(const TcInput& in, int dtype) {
  return copies_by_tile(in.p, in.stride, dtype) ? 0 : tc_result_bytes(in.rows, in.cols, dtype);
}

TcMatrix tc_operand(const TcInput& in, int dtype, void* room) {
  if (copies_by_tile(in.p, in.stride, dtype))
    return {static_cast<const bf16*>(in.p), in.rows, in.cols, in.stride, 0, 1};
  return tc_result(room, in.rows, in.cols, dtype);
}

cudaError_t launch_pack(const TcInput* in, const TcMatrix* out, int count, int dtype,
                        bool* launched, cudaStream_t stream) {
  PackJobs jobs{};
  int used = 0;
  int64_t most = 0;
  for (int i = 0; i < count; ++i) {
    if (in[i].p == nullptr || out[i].p == in[i].p || in[i].rows == 0) continue;
    jobs.job[used++] = {in[i].p, const_cast<bf16*>(out[i].p), in[i].rows, in[i].cols, in[i].stride,
                        out[i].stride, out[i].plane};
    most = std::max(most, in[i].rows * (out[i].stride / 8));
  }
  *launched = used > 0;
  if (used == 0) return cudaSuccess;
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(blocks_of(most, 256), 2368)), used);
  if (dtype == FHB_DTYPE_F32) pack_kernel<float><<<grid, 256, 0, stream>>>(jobs);
  else pack_kernel<bf16><<<grid, 256, 0, stream>>>(jobs);
  return cudaGetLastError();
}

size_t tc_factor_bytes(int64_t tokens, int64_t hidden, int dtype) {
  const int64_t places = tokens * blocks_of(hidden, kFactorGroup) * 2;
  return static_cast<size_t>(dtype == FHB_DTYPE_F32 ? places * kFactorGroup * 4
                                                    : places * kFactorGroup * 2 + round_up(places, 32));
}

TcFactors tc_factors(void* room, int64_t tokens, int64_t hidden, int dtype) {
  const int64_t groups = blocks_of(hidden, kFactorGroup), places = tokens * groups * 2;
  unsigned char* base = static_cast<unsigned char*>(room);
  return {room, dtype == FHB_DTYPE_F32 ? nullptr : base + places * kFactorGroup * 2, groups};
}

}  // namespace fhb
