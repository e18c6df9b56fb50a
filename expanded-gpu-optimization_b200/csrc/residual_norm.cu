// The RMS norms before and after a block with its gate and residual scale:
//     z = b ib wpost,  t = a r + c z,  n = t it wpre,
// with ib = 1 / sqrt(mean(b^2) + eps) and it = 1 / sqrt(mean(t^2) + eps) per row. Gradients,
// with th = t it, bh = b ib, q = dn wpre and means over the row:
//     dt = dT + it (q - th mean(q th)),   dr = a dt,   da = sum dt r,   dwpre = sum dn th,
//     dc = dt z,   dwpost = sum dt c bh,   db = ib (p - bh mean(p bh)),   p = dt c wpost.
// t is recomputed from r and b: it is not read rounded. mean(p bh) = mean(dt c z) is linear in
// mean(q th), so the backward needs one round of three row sums:
//     S1 = sum q th,   A = sum (dT + it q) c z,   B = sum th c z,
//     sum dt c z = A - it (S1 / width) B.
//
// Bound by memory: every input is read once and every output written once, a row at a time in
// registers. A row is spread over 8, 16 or 32 lanes of a warp (32 to 8 rows a CTA), or over one
// CTA, eight values a thread; a thread keeps its columns' weights, and in the backward the sums
// of its columns, from row to row. The column sums end in a second kernel, in a fixed order.
// 16,384 x 2048 with an fp32 residual, a bf16 branch and 16 gates: forward 75.5 us (402 MB, 5.3 TB/s),
// backward 121 us (604 MB, 5.0 TB/s: ten registers a value leave an SM two rows at a time, and the
// sums' barriers show), 5 us of them for the column sums. Rows wider than 4,096 have 1,024 threads, whose
// 64 registers do not hold the backward's values: it spills 0.3 KB a thread up to 8,192 and over 3 KB
// above (4,096 x 8,192 bf16: forward 61.5 us, 4.4 TB/s, backward 200 us, 2.0 TB/s; 1,600 x 20,000: 160
// and 1,160 us).
#include <algorithm>
#include <atomic>

#include "blocks.cuh"
#include "common.cuh"

namespace fhb {
namespace {


struct NormArgs {
  const void *residual, *branch, *pre_weight, *post_weight, *gate;
  int64_t rows, residual_stride, branch_stride, gate_rows;
  int width;
  const float* scale_ptr;
  float scale, eps;
  int stages;            // rows on their way to a CTA (0: it loads them itself)
  unsigned int* status;
};

// Rows on their way (a CTA a row, aligned rows): one thread starts the bulk copies of a row's
// arrays into shared memory `stages` rows ahead, so that what is in flight takes no registers.
// A stage is free again when the CTA has met in the row's sums, after everybody read it. Where a wait
// gives up (the status says so), that thread waits no more; thread 0 starts no more copies either and
// at the end waits for those on their way, since the memory is another CTA's when this one is gone.
constexpr int kMaxStages = 4;
constexpr int kMaxArrays = 5;
struct Stage {
  uint64_t* full;        // one barrier a stage
  unsigned char* base;
  int stages, at;
  uint32_t phase, bytes;  // of the arrays of one row
  bool late;              // a wait gave up
  unsigned int* status;

  __device__ __forceinline__ void start(unsigned char* memory, uint64_t* barriers, int count,
                                        uint32_t row_bytes, unsigned int* word) {
    full = barriers;
    base = memory;
    stages = count;
    at = 0;
    phase = 0;
    bytes = row_bytes;
    late = false;
    status = word;
    if (threadIdx.x == 0) {
      for (int i = 0; i < stages; ++i) mbar_init(&full[i], 1);
      fence_barrier_init();
    }
    __syncthreads();
  }
  // one thread: the arrays of a row into stage `into`
  __device__ __forceinline__ void copy(int into, const void* const (&from)[kMaxArrays],
                                       const uint32_t (&size)[kMaxArrays]) {
    if (late) return;
    mbar_arrive_expect_tx(&full[into], bytes);
    unsigned char* to = base + into * bytes;
#pragma unroll
    for (int i = 0; i < kMaxArrays; ++i)
      if (size[i] != 0) {
        bulk_copy_g2s(to, from[i], size[i], &full[into]);
        to += size[i];
      }
  }
  __device__ __forceinline__ const unsigned char* wait() {
    if (!late) late = !mbar_wait_bounded(&full[at], phase, status, FHB_STATUS_STAGE_TIMEOUT);
    return base + at * bytes;
  }
  // after the last row: whatever is still on its way has landed, or had as long again
  __device__ __forceinline__ void finish() const {
    if (threadIdx.x != 0 || !late) return;
    for (int i = 0; i < stages; ++i)
      mbar_wait_bounded(&full[i], mbar_try_wait(&full[i], 0) ? 1 : 0, status, FHB_STATUS_STAGE_TIMEOUT);
  }
  __device__ __forceinline__ void next() {
    if (++at == stages) {
      at = 0;
      phase ^= 1;
    }
  }
};

// How a row lies over threads. Lanes: 8, 16, 32 (parts of a warp, 256-thread CTAs) or 0 (the
// whole CTA, at most Most threads). V vectors of Vec values a thread. Wide: a vector is Vec (8 or
// 4) neighbours and moved in accesses of up to 16 bytes; else its values lie a row of threads apart, so that a warp's accesses
// are neighbours at any width, offset and stride.
template <int Lanes_, int Most_, int V_, int Vec_, bool Wide_>
struct Layout {
  static constexpr int Lanes = Lanes_, Most = Most_, V = V_, Vec = Vec_;
  // CTAs an SM holds in the backward
  static constexpr int Resident = Vec == 4 ? 1024 / Most : Most <= 256 ? 2 : 1;
  static constexpr bool Wide = Wide_;
  static __device__ __forceinline__ int lanes() { return Lanes ? Lanes : static_cast<int>(blockDim.x); }
  static __device__ __forceinline__ int lane() {
    return Lanes ? static_cast<int>(threadIdx.x) % Lanes : static_cast<int>(threadIdx.x);
  }
  static __device__ __forceinline__ int slots() { return Lanes ? static_cast<int>(blockDim.x) / Lanes : 1; }
  static __device__ __forceinline__ int slot() { return Lanes ? static_cast<int>(threadIdx.x) / Lanes : 0; }
  static __device__ __forceinline__ int column(int v, int i) {
    return Wide ? (v * lanes() + lane()) * Vec + i : (v * Vec + i) * lanes() + lane();
  }
};

template <typename L, typename T>
__device__ __forceinline__ void load_row(const T* row, int width, float (&x)[L::V][L::Vec]) {
#pragma unroll
  for (int v = 0; v < L::V; ++v) {
    if (L::Wide) {
      const int c = L::column(v, 0);
      if (c < width) {
        if constexpr (sizeof(T) == 2) {
          uint32_t u[L::Vec / 2];
          if constexpr (L::Vec == 8) {
            const uint4 w = *reinterpret_cast<const uint4*>(row + c);
            u[0] = w.x, u[1] = w.y, u[2] = w.z, u[3] = w.w;
          } else {
            const uint2 w = *reinterpret_cast<const uint2*>(row + c);
            u[0] = w.x, u[1] = w.y;
          }
#pragma unroll
          for (int i = 0; i < L::Vec / 2; ++i) {
            x[v][2 * i] = __uint_as_float(u[i] << 16);
            x[v][2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
          }
        } else {
#pragma unroll
          for (int i = 0; i < L::Vec / 4; ++i) {
            const float4 w = reinterpret_cast<const float4*>(row + c)[i];
            x[v][4 * i] = w.x, x[v][4 * i + 1] = w.y, x[v][4 * i + 2] = w.z, x[v][4 * i + 3] = w.w;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < L::Vec; ++i) x[v][i] = 0.0f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < L::Vec; ++i) {
        const int c = L::column(v, i);
        x[v][i] = c < width ? to_float(row[c]) : 0.0f;
      }
    }
  }
}

template <typename L, typename T>
__device__ __forceinline__ void store_row(T* row, int width, const float (&x)[L::V][L::Vec]) {
#pragma unroll
  for (int v = 0; v < L::V; ++v) {
    if (L::Wide) {
      const int c = L::column(v, 0);
      if (c >= width) continue;
      if constexpr (sizeof(T) == 2) {
        uint32_t u[L::Vec / 2];
#pragma unroll
        for (int i = 0; i < L::Vec / 2; ++i)
          asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u[i]) : "f"(x[v][2 * i + 1]), "f"(x[v][2 * i]));
        if constexpr (L::Vec == 8)
          *reinterpret_cast<uint4*>(row + c) = make_uint4(u[0], u[1], u[2], u[3]);
        else
          *reinterpret_cast<uint2*>(row + c) = make_uint2(u[0], u[1]);
      } else {
#pragma unroll
        for (int i = 0; i < L::Vec / 4; ++i)
          reinterpret_cast<float4*>(row + c)[i] =
              make_float4(x[v][4 * i], x[v][4 * i + 1], x[v][4 * i + 2], x[v][4 * i + 3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < L::Vec; ++i) {
        const int c = L::column(v, i);
        if (c < width) row[c] = from_float<T>(x[v][i]);
      }
    }
  }
}

template <typename L>
__device__ __forceinline__ void fill(float (&x)[L::V][L::Vec], float value) {
#pragma unroll
  for (int v = 0; v < L::V; ++v)
#pragma unroll
    for (int i = 0; i < L::Vec; ++i) x[v][i] = value;
}

// Sums of K values over the threads of a row, in a fixed order, to all of them. `round` flips
// between calls: two buffers need one barrier a call.
template <typename L, int K>
__device__ __forceinline__ void row_sum(float (&s)[K], int& round) {
  constexpr int kFirst = L::Lanes ? L::Lanes / 2 : 16;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int m = kFirst; m >= 1; m >>= 1) s[k] += __shfl_xor_sync(0xffffffffu, s[k], m);
  if (L::Lanes) return;
  __shared__ float part[2][K][32];
  const int warps = static_cast<int>(blockDim.x) / 32;
  if (threadIdx.x % 32 == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) part[round][k][threadIdx.x / 32] = s[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int lane = static_cast<int>(threadIdx.x) % 32;
    s[k] = lane < warps ? part[round][k][lane] : 0.0f;
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) s[k] += __shfl_xor_sync(0xffffffffu, s[k], m);
  }
  round ^= 1;
}

// A row's value where the row exists: rows of a warp's other slots take part in its shuffles.
#define FHB_EACH(L) \
  _Pragma("unroll") for (int v = 0; v < L::V; ++v) _Pragma("unroll") for (int i = 0; i < L::Vec; ++i)

template <typename L, typename TR, typename T, bool Staged>
__global__ void __launch_bounds__(L::Most, L::Most <= 256 ? 4 : 1)
    norm_kernel(NormArgs a, TR* __restrict__ total, T* __restrict__ normed,
                float* __restrict__ stats) {
  const float scale = a.scale_ptr != nullptr ? *a.scale_ptr : a.scale;
  const float inverse = 1.0f / static_cast<float>(a.width);
  const bool post = a.post_weight != nullptr, gated = a.gate != nullptr;
  const bool one_gate = gated && a.gate_rows >= a.rows;
  float wpre[L::V][L::Vec], wpost[L::V][L::Vec], gate[L::V][L::Vec];
  load_row<L>(static_cast<const T*>(a.pre_weight), a.width, wpre);
  // what is not there is 1: no value's arithmetic branches
  fill<L>(wpost, 1.0f);
  fill<L>(gate, 1.0f);
  if (post) load_row<L>(static_cast<const T*>(a.post_weight), a.width, wpost);
  if (one_gate) load_row<L>(static_cast<const T*>(a.gate), a.width, gate);
  int round = 0;
  const int64_t step = static_cast<int64_t>(gridDim.x) * L::slots();
  const auto residual_at = [&](int64_t row) {
    return static_cast<const TR*>(a.residual) + row * a.residual_stride;
  };
  const auto branch_at = [&](int64_t row) {
    return static_cast<const T*>(a.branch) + row * a.branch_stride;
  };
  const auto gate_at = [&](int64_t row) {
    return static_cast<const T*>(a.gate) + row / a.gate_rows * a.width;
  };
  extern __shared__ __align__(16) unsigned char rows_memory[];
  __shared__ uint64_t full[kMaxStages];
  Stage stage;
  const uint32_t wide = a.width * sizeof(TR), narrow = a.width * sizeof(T);
  const uint32_t size[kMaxArrays] = {wide, a.branch != nullptr ? narrow : 0,
                                     gated && !one_gate ? narrow : 0, 0, 0};
  const auto send = [&](int into, int64_t row) {
    const void* const from[kMaxArrays] = {residual_at(row), branch_at(row),
                                          gated ? gate_at(row) : nullptr, nullptr, nullptr};
    stage.copy(into, from, size);
  };
  if (Staged) {
    stage.start(rows_memory, full, a.stages, size[0] + size[1] + size[2], a.status);
    if (threadIdx.x == 0)
      for (int i = 0; i < a.stages && blockIdx.x + i * step < a.rows; ++i) send(i, blockIdx.x + i * step);
  }
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * L::slots(); first < a.rows; first += step) {
    const int64_t row = first + L::slot();
    const bool real = row < a.rows;
    float t[L::V][L::Vec], b[L::V][L::Vec];
    fill<L>(b, 0.0f);
    if (Staged) {
      const unsigned char* from = stage.wait();
      load_row<L>(reinterpret_cast<const TR*>(from), a.width, t);
      if (size[1] != 0) load_row<L>(reinterpret_cast<const T*>(from + size[0]), a.width, b);
      if (size[2] != 0) load_row<L>(reinterpret_cast<const T*>(from + size[0] + size[1]), a.width, gate);
    } else {
      fill<L>(t, 0.0f);
      if (real) {
        load_row<L>(residual_at(row), a.width, t);
        if (a.branch != nullptr) load_row<L>(branch_at(row), a.width, b);
        if (gated && !one_gate) load_row<L>(gate_at(row), a.width, gate);
      }
    }
    float ib = 1.0f;
    if (post) {
      float s[1] = {};
      FHB_EACH(L) s[0] += b[v][i] * b[v][i];
      row_sum<L>(s, round);
      ib = 1.0f / sqrtf(s[0] * inverse + a.eps);
    }
    float s[1] = {};
    FHB_EACH(L) {
      t[v][i] = scale * t[v][i] + b[v][i] * ib * wpost[v][i] * gate[v][i];
      s[0] += t[v][i] * t[v][i];
    }
    row_sum<L>(s, round);
    if (Staged) {
      const int64_t ahead = row + a.stages * step;
      if (threadIdx.x == 0 && ahead < a.rows) send(stage.at, ahead);
      stage.next();
    }
    const float it = 1.0f / sqrtf(s[0] * inverse + a.eps);
    if (!real) continue;
    if (total != nullptr) store_row<L>(total + row * a.width, a.width, t);
    FHB_EACH(L) t[v][i] = t[v][i] * it * wpre[v][i];
    store_row<L>(normed + row * a.width, a.width, t);
    if (stats != nullptr && L::lane() == 0) {
      stats[2 * row] = ib;
      stats[2 * row + 1] = it;
    }
  }
  if (Staged) stage.finish();
}

// ---- backward ----
// Rows are cut into units: `parts` equal parts of every gate group (of all rows without a gate
// or with one per channel). A slot takes whole units, so a group's sum over its rows is made
// from at most `parts` pieces.
struct Units {
  int groups, group_rows, parts, part_rows, slots, grid;  // at most 2^30 rows
};
struct NormGrads {
  const void *total, *normed;
  int64_t total_stride, normed_stride;
  void *residual, *branch, *gate;  // gate: groups of one part, written here
  float* columns;      // [grid][3][width]: sums for dwpre, dwpost, dgate (one per channel)
  float* gate_parts;   // [group][part][width] where groups have several parts
  float* scale_parts;  // [grid]
  bool want_pre, want_post, want_gate, want_scale;
};

template <typename L, typename TR, typename T, bool Staged>
__global__ void __launch_bounds__(L::Most, L::Resident)
    norm_backward_kernel(NormArgs a, NormGrads g, Units units, const float* __restrict__ stats) {
  const float scale = a.scale_ptr != nullptr ? *a.scale_ptr : a.scale;
  const float inverse = 1.0f / static_cast<float>(a.width);
  const bool post = a.post_weight != nullptr, gated = a.gate != nullptr, branch = a.branch != nullptr;
  const bool by_group = gated && units.groups > 1;
  float wpre[L::V][L::Vec], wpost[L::V][L::Vec], gate[L::V][L::Vec];
  load_row<L>(static_cast<const T*>(a.pre_weight), a.width, wpre);
  // what is not there is 1: no value's arithmetic branches
  fill<L>(wpost, 1.0f);
  fill<L>(gate, 1.0f);
  if (post) load_row<L>(static_cast<const T*>(a.post_weight), a.width, wpost);
  if (gated) load_row<L>(static_cast<const T*>(a.gate), a.width, gate);
  float spre[L::V][L::Vec], spost[L::V][L::Vec], sgate[L::V][L::Vec], sscale = 0.0f;
  fill<L>(spre, 0.0f);
  fill<L>(spost, 0.0f);
  fill<L>(sgate, 0.0f);
  int round = 0;
  const int count = units.groups * units.parts, rows = static_cast<int>(a.rows);
  const int step = static_cast<int>(gridDim.x) * L::slots();
  // the rows [begin, end) of a unit, none for a unit past the last
  const auto rows_of = [&](int unit, int& begin, int& end) {
    const int group = unit / units.parts, part = unit - group * units.parts;
    const int first = group * units.group_rows;
    begin = first + part * units.part_rows;
    end = unit < count ? min(begin + units.part_rows, min(rows - first, units.group_rows) + first) : begin;
  };
  extern __shared__ __align__(16) unsigned char rows_memory[];
  __shared__ uint64_t full[kMaxStages];
  Stage stage;
  const uint32_t wide = a.width * sizeof(TR), narrow = a.width * sizeof(T);
  const uint32_t size[kMaxArrays] = {wide, branch ? narrow : 0, g.total != nullptr ? wide : 0,
                                     g.normed != nullptr ? narrow : 0, by_group ? narrow : 0};
  // thread 0's place in the rows to come
  int send_unit = blockIdx.x, send_row = 0, send_end = 0;
  const auto send = [&](int into) {
    while (send_row >= send_end) {
      if (send_unit >= count) return;
      rows_of(send_unit, send_row, send_end);
      send_unit += step;
    }
    const void* const from[kMaxArrays] = {
        static_cast<const TR*>(a.residual) + static_cast<int64_t>(send_row) * a.residual_stride,
        static_cast<const T*>(a.branch) + static_cast<int64_t>(send_row) * a.branch_stride,
        static_cast<const TR*>(g.total) + static_cast<int64_t>(send_row) * g.total_stride,
        static_cast<const T*>(g.normed) + static_cast<int64_t>(send_row) * g.normed_stride,
        static_cast<const T*>(a.gate) + static_cast<int64_t>(send_row / units.group_rows) * a.width};
    stage.copy(into, from, size);
    ++send_row;
  };
  if (Staged) {
    stage.start(rows_memory, full, a.stages, size[0] + size[1] + size[2] + size[3] + size[4], a.status);
    if (threadIdx.x == 0)
      for (int i = 0; i < a.stages; ++i) send(i);
  }
  for (int first = static_cast<int>(blockIdx.x) * L::slots(); first < count; first += step) {
    const int unit = first + L::slot();
    int begin, end;
    rows_of(unit, begin, end);
    if (!Staged && by_group && unit < count)
      load_row<L>(static_cast<const T*>(a.gate) + static_cast<int64_t>(unit / units.parts) * a.width, a.width, gate);
    // the slots of a warp go through as many rows together, some of them without a row
    for (int k = 0; k < units.part_rows; ++k) {
      const int64_t row = begin + k;
      const bool real = row < end;
      if (L::Lanes == 0 && !real) break;
      float r[L::V][L::Vec], b[L::V][L::Vec], dT[L::V][L::Vec], dn[L::V][L::Vec];
      float ib = 1.0f, it = 1.0f;
      if (real) {
        ib = stats[2 * row];
        it = stats[2 * row + 1];
      }
      fill<L>(b, 0.0f);
      fill<L>(dT, 0.0f);
      fill<L>(dn, 0.0f);
      if (Staged) {
        const unsigned char* from = stage.wait();
        load_row<L>(reinterpret_cast<const TR*>(from), a.width, r);
        from += size[0];
        if (size[1] != 0) load_row<L>(reinterpret_cast<const T*>(from), a.width, b);
        from += size[1];
        if (size[2] != 0) load_row<L>(reinterpret_cast<const TR*>(from), a.width, dT);
        from += size[2];
        if (size[3] != 0) load_row<L>(reinterpret_cast<const T*>(from), a.width, dn);
        from += size[3];
        if (size[4] != 0) load_row<L>(reinterpret_cast<const T*>(from), a.width, gate);
      } else {
        fill<L>(r, 0.0f);
        if (real) {
          load_row<L>(static_cast<const TR*>(a.residual) + row * a.residual_stride, a.width, r);
          if (branch) load_row<L>(static_cast<const T*>(a.branch) + row * a.branch_stride, a.width, b);
          if (g.total != nullptr)
            load_row<L>(static_cast<const TR*>(g.total) + row * g.total_stride, a.width, dT);
          if (g.normed != nullptr)
            load_row<L>(static_cast<const T*>(g.normed) + row * g.normed_stride, a.width, dn);
        }
      }
      float s[3] = {};
      FHB_EACH(L) {
        const float cz = b[v][i] * ib * wpost[v][i] * gate[v][i];
        const float th = (scale * r[v][i] + cz) * it, q = dn[v][i] * wpre[v][i];
        s[0] += q * th;
        s[1] += (dT[v][i] + it * q) * cz;
        s[2] += th * cz;
      }
      row_sum<L>(s, round);
      if (Staged) {
        if (threadIdx.x == 0) send(stage.at);
        stage.next();
      }
      if (!real) continue;
      const float m1 = s[0] * inverse, m2 = post ? (s[1] - it * m1 * s[2]) * inverse : 0.0f;
      FHB_EACH(L) {
        const float bh = b[v][i] * ib, z = bh * wpost[v][i], cz = z * gate[v][i];
        const float th = (scale * r[v][i] + cz) * it, q = dn[v][i] * wpre[v][i];
        const float dt = dT[v][i] + it * (q - th * m1);
        const float dz = dt * gate[v][i];
        spre[v][i] += dn[v][i] * th;
        spost[v][i] += dz * bh;
        sgate[v][i] += dt * z;
        sscale += dt * r[v][i];
        r[v][i] = scale * dt;
        b[v][i] = ib * (dz * wpost[v][i] - bh * m2);
      }
      if (g.residual != nullptr) store_row<L>(static_cast<TR*>(g.residual) + row * a.width, a.width, r);
      if (g.branch != nullptr) store_row<L>(static_cast<T*>(g.branch) + row * a.width, a.width, b);
    }
    if (by_group) {
      if (unit < count && g.want_gate) {
        if (units.parts == 1)
          store_row<L>(static_cast<T*>(g.gate) + static_cast<int64_t>(unit) * a.width, a.width, sgate);
        else
          FHB_EACH(L) {
            const int c = L::column(v, i);
            if (c < a.width) g.gate_parts[static_cast<int64_t>(unit) * a.width + c] = sgate[v][i];
          }
      }
      fill<L>(sgate, 0.0f);
    }
  }
  if (Staged) stage.finish();
  // the CTA's column sums: its slots' one after the other
  float* columns = reinterpret_cast<float*>(rows_memory);
  float* out = g.columns + static_cast<int64_t>(blockIdx.x) * 3 * a.width;
  const auto leave = [&](const float (&x)[L::V][L::Vec], int which) {
    if (L::Lanes == 0) {
      FHB_EACH(L) {
        const int c = L::column(v, i);
        if (c < a.width) out[which * a.width + c] = x[v][i];
      }
      return;
    }
    __syncthreads();
    FHB_EACH(L) {
      const int c = L::column(v, i);
      if (c < a.width) columns[L::slot() * a.width + c] = x[v][i];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.width; c += blockDim.x) {
      float sum = 0.0f;
      for (int k = 0; k < L::slots(); ++k) sum += columns[k * a.width + c];
      out[which * a.width + c] = sum;
    }
  };
  if (g.want_pre) leave(spre, 0);
  if (g.want_post) leave(spost, 1);
  if (g.want_gate && !by_group) leave(sgate, 2);
  if (g.want_scale) {
    float s[1] = {sscale};
    row_sum<L>(s, round);
    __shared__ float by_slot[32];
    __syncthreads();
    if (L::lane() == 0) by_slot[L::slot()] = s[0];
    __syncthreads();
    if (threadIdx.x == 0) {
      float sum = 0.0f;
      for (int k = 0; k < L::slots(); ++k) sum += by_slot[k];
      g.scale_parts[blockIdx.x] = sum;
    }
  }
}

// Second kernel of the column sums: out[c] = the rows in[k * stride + c] in a fixed order. One
// task per blockIdx.y: dwpre, dwpost, dgate of all rows; the scale; then the gate groups.
struct Totals {
  const float* columns;
  const float* gate_parts;
  const float* scale_parts;
  int64_t grid, parts, width;
  void *pre, *post, *gate;
  float* scale;
  bool by_group;
};
template <typename T>
__global__ void __launch_bounds__(256) norm_totals_kernel(Totals t) {
  const int64_t task = blockIdx.y;
  const int lane = threadIdx.x % 32, group = threadIdx.x / 32;
  if (task == 3) {
    if (blockIdx.x != 0 || t.scale == nullptr) return;
    __shared__ double by_thread[256];
    double s = 0.0;
    for (int64_t k = threadIdx.x; k < t.grid; k += 256) s += t.scale_parts[k];
    by_thread[threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      s = 0.0;
      for (int k = 0; k < 256; ++k) s += by_thread[k];
      *t.scale = static_cast<float>(s);
    }
    return;
  }
  const float* in;
  int64_t rows, stride;
  T* out;
  if (task < 3) {
    in = t.columns + task * t.width;
    rows = t.grid;
    stride = 3 * t.width;
    out = static_cast<T*>(task == 0 ? t.pre : task == 1 ? t.post : t.by_group ? nullptr : t.gate);
  } else {
    in = t.gate_parts + (task - 4) * t.parts * t.width;
    rows = t.parts;
    stride = t.width;
    out = static_cast<T*>(t.gate) + (task - 4) * t.width;
  }
  if (out == nullptr) return;
  __shared__ float by_group[8][32];
  const int64_t c = blockIdx.x * 32ll + lane;
  float s = 0.0f;
  if (c < t.width) {
    int64_t k = group;
    for (; k + 56 < rows; k += 64) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = in[(k + 8 * j) * stride + c];
#pragma unroll
      for (int j = 0; j < 8; ++j) s += v[j];
    }
    for (; k < rows; k += 8) s += in[k * stride + c];
  }
  by_group[group][lane] = s;
  __syncthreads();
  if (group == 0 && c < t.width) {
    s = 0.0f;
    for (int k = 0; k < 8; ++k) s += by_group[k][lane];
    out[c] = from_float<T>(s);
  }
}

// Test hook: three rows of 1 KB on their way, of which the first is said to be longer than it is, so
// that the wait for it gives up. out: whether it did; which of the three have landed by then, as bits;
// whether a row started after it lands.
__global__ void staged_wait_selftest_kernel(const float* rows, float* out, unsigned int* status) {
  constexpr int kRowBytes = 1024, kCount = 3;
  __shared__ __align__(16) unsigned char memory[kCount * kRowBytes];
  __shared__ uint64_t full[kMaxStages];
  const uint32_t size[kMaxArrays] = {kRowBytes, 0, 0, 0, 0};
  Stage stage;
  stage.start(memory, full, kCount, kRowBytes, status);
  const auto send = [&](int into) {
    const void* const from[kMaxArrays] = {rows + into * (kRowBytes / 4), nullptr, nullptr, nullptr, nullptr};
    stage.copy(into, from, size);
  };
  if (threadIdx.x == 0)
    for (int i = 0; i < kCount; ++i) {
      stage.bytes = kRowBytes + (i == 0 ? 16 : 0);
      send(i);
    }
  stage.bytes = kRowBytes;
  stage.wait();
  stage.finish();
  if (threadIdx.x == 0) {
    int landed = 0;
    for (int i = 0; i < kCount; ++i) landed |= (mbar_try_wait(&full[i], 0) ? 1 : 0) << i;
    out[0] = stage.late ? 1.0f : 0.0f;
    out[1] = static_cast<float>(landed);
    send(1);
    bool more = false;
    for (int i = 0; i < 10; ++i) more = more || mbar_try_wait_for(&full[1], 1, kSuspendHintNs);
    out[2] = more ? 1.0f : 0.0f;
  }
}

// ---- launches ----
NormArgs arguments(const fhb_norm_problem& p) {
  return {p.residual, p.branch, p.pre_weight, p.post_weight, p.gate, p.rows, p.residual_stride,
          p.branch_stride, p.gate != nullptr ? p.gate_rows : std::max<int64_t>(p.rows, 1),
          static_cast<int>(p.width), p.residual_scale_ptr, p.residual_scale, p.eps, 0, nullptr};
}

// Rows a CTA can have on their way in its part of an SM's shared memory; fewer than two: none.
constexpr int kStagedBytes = 216 * 1024;  // of an SM
int stages_of(int64_t row_bytes, int resident) {
  const int64_t n = std::min<int64_t>(kStagedBytes / resident / row_bytes, kMaxStages);
  return n >= 2 ? static_cast<int>(n) : 0;
}

bool wide_rows(const void* p, int64_t stride, int dtype) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 &&
         stride * static_cast<int64_t>(dtype_bytes(dtype)) % 16 == 0;
}
bool wide_inputs(const fhb_norm_problem& p) {
  return p.width % 8 == 0 && wide_rows(p.residual, p.residual_stride, p.residual_dtype) &&
         wide_rows(p.branch, p.branch_stride, p.dtype) && wide_rows(p.pre_weight, 0, p.dtype) &&
         wide_rows(p.post_weight, 0, p.dtype) && wide_rows(p.gate, p.width, p.dtype);
}

// Threads of a row: a power of 2, at most 1,024. 8 values each (rows wider than 8,192 take four
// vectors a thread); 4 each in the backward of unaligned rows, which loads them itself: more
// warps then hide it (30,000 x 777: 317 -> 174 us), while aligned rows, which come by bulk
// copies, need the registers more (16,384 x 2048: 1.6 times the time with 4 values).
int vector_of(int64_t width, bool backward, bool wide) {
  return backward && !wide && width > 256 && width <= 4096 ? 4 : 8;
}
int row_threads(int64_t width, bool backward, bool wide) {
  const int vector = vector_of(width, backward, wide);
  const int64_t need = (width + vector - 1) / vector;
  int n = 8;
  while (n < need && n < 1024) n *= 2;
  return n;
}
int slots_of(int threads) { return threads <= 32 ? 256 / threads : 1; }
int block_of(int threads) { return threads <= 32 ? 256 : threads; }

// CTAs an SM holds (Layout::Resident in the backward, whose sums take registers).
int resident_of(int64_t width, bool backward, bool wide) {
  const int threads = row_threads(width, backward, wide), block = block_of(threads);
  if (!backward) return block <= 256 ? 4 : 1;
  if (vector_of(width, true, wide) == 4) return block <= 256 ? 4 : block <= 512 ? 2 : 1;
  return block <= 256 ? 2 : 1;
}
int64_t ctas(int64_t width, bool backward, bool wide, const DeviceInfo& dev) {
  return static_cast<int64_t>(dev.sms) * resident_of(width, backward, wide);
}

Units units_of(const fhb_norm_problem& p, bool wide, const DeviceInfo& dev) {
  const int threads = row_threads(p.width, true, wide);
  const int64_t rows = std::max<int64_t>(p.rows, 1);
  const int64_t group_rows = p.gate != nullptr ? std::min(p.gate_rows, rows) : rows;
  const int64_t groups = (rows + group_rows - 1) / group_rows;
  const int64_t most = ctas(p.width, true, wide, dev), slots = most * slots_of(threads);
  int64_t parts = std::min(std::max<int64_t>(1, slots / groups), group_rows);
  const int64_t part_rows = (group_rows + parts - 1) / parts;
  parts = (group_rows + part_rows - 1) / part_rows;
  const int64_t grid = std::min((groups * parts + slots_of(threads) - 1) / slots_of(threads), most);
  return {static_cast<int>(groups), static_cast<int>(group_rows), static_cast<int>(parts),
          static_cast<int>(part_rows), static_cast<int>(slots), static_cast<int>(grid)};
}

// Calls body(Layout) with the layout for the width.
template <bool Wide, bool Backward, typename Body>
cudaError_t with_layout(int64_t width, Body body) {
  if (width > 8192) return body(Layout<0, 1024, 4, 8, Wide>{});
  const int threads = row_threads(width, Backward, Wide);
  if constexpr (Backward && !Wide) {
    if (vector_of(width, true, false) == 4) {
      if (threads <= 256) return body(Layout<0, 256, 1, 4, Wide>{});
      if (threads <= 512) return body(Layout<0, 512, 1, 4, Wide>{});
      return body(Layout<0, 1024, 1, 4, Wide>{});
    }
  }
  if (threads == 8) return body(Layout<8, 256, 1, 8, Wide>{});
  if (threads == 16) return body(Layout<16, 256, 1, 8, Wide>{});
  if (threads == 32) return body(Layout<32, 256, 1, 8, Wide>{});
  if constexpr (!Backward || Wide) {
    if (threads <= 256) return body(Layout<0, 256, 1, 8, Wide>{});
    if (threads <= 512) return body(Layout<0, 512, 1, 8, Wide>{});
  }
  return body(Layout<0, 1024, 1, 8, Wide>{});
}
template <bool Backward, typename Body>
cudaError_t with_layout(bool wide, int64_t width, Body body) {
  return wide ? with_layout<true, Backward>(width, body) : with_layout<false, Backward>(width, body);
}

// The most shared memory that a launch of a staged kernel asks for, set with its first call on a
// device: the limit is the kernel's, not the launch's, and host threads with rows of different bytes
// share it. (All of these kernels at once would take 18 ms to load.)
template <bool Backward, typename L, typename TR, typename T>
cudaError_t allow_staged() {
  static std::atomic<uint64_t> allowed{0};  // a bit a device
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const uint64_t bit = uint64_t{1} << (device % 64);
  if ((allowed.load(std::memory_order_acquire) & bit) != 0) return cudaSuccess;
  if constexpr (Backward)
    e = cudaFuncSetAttribute(norm_backward_kernel<L, TR, T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kStagedBytes / L::Resident);
  else
    e = cudaFuncSetAttribute(norm_kernel<L, TR, T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kStagedBytes / (L::Most <= 256 ? 4 : 1));
  if (e == cudaSuccess) allowed.fetch_or(bit, std::memory_order_release);
  return e;
}

template <typename TR, typename T>
cudaError_t forward(const fhb_norm_problem& p, void* total, void* normed, float* stats,
                    const DeviceInfo& dev, cudaStream_t stream) {
  const bool wide = wide_inputs(p) && wide_rows(total, p.width, p.residual_dtype) &&
                    wide_rows(normed, p.width, p.dtype);
  const int threads = row_threads(p.width, false, wide);
  const int64_t need = (p.rows + slots_of(threads) - 1) / slots_of(threads);
  const unsigned grid = static_cast<unsigned>(std::min(need, ctas(p.width, false, wide, dev)));
  NormArgs args = arguments(p);
  const int64_t row_bytes =
      p.width * (sizeof(TR) + (p.branch != nullptr ? sizeof(T) : 0) +
                 (p.gate != nullptr && p.gate_rows < p.rows ? sizeof(T) : 0));
  // a single row a CTA has nothing to fetch ahead
  if (threads > 32 && wide && need > grid) args.stages = stages_of(row_bytes, resident_of(p.width, false, wide));
  args.status = dev.status;
  return with_layout<false>(wide, p.width, [&](auto layout) {
    using L = decltype(layout);
    if constexpr (L::Lanes == 0 && L::Wide)
      if (args.stages > 0) {
        const cudaError_t e = allow_staged<false, L, TR, T>();
        if (e != cudaSuccess) return e;
        norm_kernel<L, TR, T, true><<<grid, block_of(threads), args.stages * row_bytes, stream>>>(
            args, static_cast<TR*>(total), static_cast<T*>(normed), stats);
        return cudaGetLastError();
      }
    norm_kernel<L, TR, T, false><<<grid, block_of(threads), 0, stream>>>(
        args, static_cast<TR*>(total), static_cast<T*>(normed), stats);
    return cudaGetLastError();
  });
}

struct Room {
  float *columns, *gate_parts, *scale_parts;
  size_t bytes;
};
Room room_of(const fhb_norm_problem& p, const Units& u, void* base) {
  float* at = static_cast<float*>(base);
  const auto padded = [](int64_t n) { return (n + 31) / 32 * 32; };
  const int64_t columns = padded(u.grid * 3ll * p.width);
  const int64_t gates = u.groups > 1 && u.parts > 1 ? padded(static_cast<int64_t>(u.groups) * u.parts * p.width) : 0;
  return {at, at + columns, at + columns + gates,
          static_cast<size_t>(columns + gates + padded(u.grid)) * 4};
}

template <typename TR, typename T>
cudaError_t backward(const fhb_norm_problem& p, const NormGrads& g, const Units& u, const Totals& t,
                     const float* stats, bool wide, const DeviceInfo& dev,
                     cudaStream_t stream) {
  const int threads = row_threads(p.width, true, wide);
  const size_t smem = threads <= 32 ? static_cast<size_t>(slots_of(threads)) * p.width * 4 : 0;
  NormArgs args = arguments(p);
  const int64_t row_bytes = p.width * (sizeof(TR) + (p.branch != nullptr ? sizeof(T) : 0) +
                                       (g.total != nullptr ? sizeof(TR) : 0) +
                                       (g.normed != nullptr ? sizeof(T) : 0) +
                                       (p.gate != nullptr && u.groups > 1 ? sizeof(T) : 0));
  if (threads > 32 && wide && p.rows > u.grid) args.stages = stages_of(row_bytes, resident_of(p.width, true, wide));
  args.status = dev.status;
  const cudaError_t e = with_layout<true>(wide, p.width, [&](auto layout) {
    using L = decltype(layout);
    if constexpr (L::Lanes == 0 && L::Wide)
      if (args.stages > 0) {
        const cudaError_t allowed = allow_staged<true, L, TR, T>();
        if (allowed != cudaSuccess) return allowed;
        norm_backward_kernel<L, TR, T, true>
            <<<static_cast<unsigned>(u.grid), block_of(threads), args.stages * row_bytes, stream>>>(args, g, u, stats);
        return cudaGetLastError();
      }
    norm_backward_kernel<L, TR, T, false>
        <<<static_cast<unsigned>(u.grid), block_of(threads), smem, stream>>>(args, g, u, stats);
    return cudaGetLastError();
  });
  if (e != cudaSuccess || !(g.want_pre || g.want_post || g.want_gate || g.want_scale)) return e;
  const bool groups = t.by_group && g.want_gate && u.parts > 1;
  const dim3 grid(static_cast<unsigned>((p.width + 31) / 32), static_cast<unsigned>(4 + (groups ? u.groups : 0)));
  norm_totals_kernel<T><<<grid, 256, 0, stream>>>(t);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_residual_norm(const fhb_norm_problem& p, void* total, void* normed,
                                 float* stats, const DeviceInfo& dev, cudaStream_t stream) {
  if (p.residual_dtype == FHB_DTYPE_F32)
    return p.dtype == FHB_DTYPE_F32 ? forward<float, float>(p, total, normed, stats, dev, stream)
                                    : forward<float, bf16>(p, total, normed, stats, dev, stream);
  return forward<bf16, bf16>(p, total, normed, stats, dev, stream);
}

cudaError_t launch_staged_wait_selftest(const float* rows, float* out, const DeviceInfo& dev,
                                        cudaStream_t stream) {
  staged_wait_selftest_kernel<<<1, 64, 0, stream>>>(rows, out, dev.status);
  return cudaGetLastError();
}

size_t residual_norm_workspace_bytes(const fhb_norm_problem& p, const DeviceInfo& dev) {
  // whether the gradients' rows are aligned is not known yet
  return std::max(room_of(p, units_of(p, true, dev), nullptr).bytes,
                  room_of(p, units_of(p, false, dev), nullptr).bytes);
}

cudaError_t launch_residual_norm_backward(const fhb_norm_problem& p, const void* grad_total,
                                          int64_t grad_total_stride, const void* grad_normed,
                                          int64_t grad_normed_stride, const float* stats,
                                          const fhb_norm_grads& out, void* workspace,
                                          const DeviceInfo& dev, cudaStream_t stream) {
  const bool wide = wide_inputs(p) && wide_rows(grad_total, grad_total_stride, p.residual_dtype) &&
                    wide_rows(grad_normed, grad_normed_stride, p.dtype) &&
                    wide_rows(out.residual, p.width, p.residual_dtype) &&
                    wide_rows(out.branch, p.width, p.dtype) && wide_rows(out.gate, p.width, p.dtype);
  const Units u = units_of(p, wide, dev);
  const Room room = room_of(p, u, workspace);
  const NormGrads g{grad_total, grad_normed, grad_total_stride, grad_normed_stride, out.residual,
                    out.branch, out.gate, room.columns, room.gate_parts, room.scale_parts,
                    out.pre_weight != nullptr, out.post_weight != nullptr, out.gate != nullptr,
                    out.residual_scale != nullptr};
  const Totals t{room.columns, room.gate_parts, room.scale_parts, u.grid, u.parts, p.width,
                 out.pre_weight, out.post_weight, out.gate, out.residual_scale,
                 p.gate != nullptr && u.groups > 1};
  if (p.residual_dtype == FHB_DTYPE_F32)
    return p.dtype == FHB_DTYPE_F32 ? backward<float, float>(p, g, u, t, stats, wide, dev, stream)
                                    : backward<float, bf16>(p, g, u, t, stats, wide, dev, stream);
  return backward<bf16, bf16>(p, g, u, t, stats, wide, dev, stream);
}

}  // namespace fhb
