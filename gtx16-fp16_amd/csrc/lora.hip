// Low-rank adapters of many requests beside one linear layer (g16_lora_*; formulas in g16.h):
//   low[m, :] = scale[a] * x[m, :] @ down[a]^T,   out[m, :] = y[m, :] + low[m, :] @ up[a]^T,   a = index[m],
// where y is the shared projection's result.
//
// Both products work on tiles of 16 rows on the 16x16 MFMA blocks, one adapter at a time, for whichever
// rows of the tile have it; the rows of a tile are looked at once (a ballot per adapter among them), so
// they may come in any order and need no sorting. fp32 activations, and the second product, whose left
// side is fp32 sums, run on v_mfma_f32_16x16x4_f32, so nothing is rounded on the way to the output.
// A tile's adapters may be dealt to several workgroups (`slots`): their rows are disjoint, so nothing has
// to be added across them. Decode batches, where every row has its own adapter, are bound by reading the
// adapters (rank * (K + N) * 2 bytes each) and need the parallel loads.
#include "g16_common.hpp"

namespace g16 {
namespace {

typedef float float8v __attribute__((ext_vector_type(8)));

constexpr int kRows = 16;  // rows of a tile
constexpr int kThreads = 256, kWaves = 4;

__device__ inline float4v mma16(half8 a, half8 b, float4v c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ inline float4v mma16(float8v a, float8v b, float4v c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
  return c;
}
__device__ inline float8v widen(half8 h) { return __builtin_convertvector(h, float8v); }
__device__ inline half8 as_operand(half8 h, _Float16) { return h; }
__device__ inline float8v as_operand(half8 h, float) { return widen(h); }

template <typename T>
struct Vec8 {
  using V = half8;
};
template <>
struct Vec8<float> {
  using V = float8v;
};

struct Params {
  const void* x;
  const _Float16 *down, *up;
  const int32_t* index;
  const float *scale, *y;
  void* out;
  float* low;  // [splits][M][rank]
  int M, K, N, rank, adapters, slots, splits;
};

// Calls f(adapter, rows) for every `slots`-th adapter (from `slot` on) among the tile's rows; rows: bit i
// for row i. `mine` is the adapter of row lane % 16, negative for none.
template <typename F>
__device__ inline void each_adapter(int mine, int slot, int slots, const F& f) {
  uint32_t left = static_cast<uint32_t>(__ballot(mine >= 0)) & 0xffffu;
  for (int i = 0; left != 0; ++i) {
    const int a = __builtin_amdgcn_readlane(mine, __builtin_ctz(left));
    const uint32_t rows = static_cast<uint32_t>(__ballot(mine == a)) & 0xffffu;
    left &= ~rows;
    if (i % slots == slot) f(a, rows);
  }
}

__device__ inline int adapter_of(const Params& p, int row) {
  const int a = row < p.M ? p.index[row] : -1;
  return a < p.adapters ? a : -1;
}

// low: split blockIdx.y of K, a quarter of it to each wavefront; RB blocks of 16 rank columns.
template <typename T, int RB>
__global__ __launch_bounds__(kThreads) void shrink_kernel(Params p) {
  __shared__ float4v part[kWaves][RB][kWave];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int slot = blockIdx.x % p.slots, m0 = static_cast<int>(blockIdx.x / p.slots) * kRows, split = blockIdx.y;
  const int mine = adapter_of(p, m0 + (lane & 15));
  const int steps = ceil_div(p.K, 32), parts = p.splits * kWaves, at = split * kWaves + wave;
  const int s0 = static_cast<int>(static_cast<int64_t>(steps) * at / parts), s1 = static_cast<int>(static_cast<int64_t>(steps) * (at + 1) / parts);
  const int kl = (lane >> 4) * 8;
  const T* xrow = static_cast<const T*>(p.x) + static_cast<size_t>(min(m0 + (lane & 15), p.M - 1)) * p.K;
  each_adapter(mine, slot, p.slots, [&](int a, uint32_t rows) {
    const _Float16* drow = p.down + (static_cast<size_t>(a) * p.rank + (lane & 15)) * p.K;
    float4v acc[RB] = {};
#pragma unroll 4
    for (int s = s0; s < s1; ++s) {
      const int k = s * 32 + kl;
      typename Vec8<T>::V xv = {};
      half8 dv[RB] = {};
      if (k < p.K) {
        xv = *reinterpret_cast<const typename Vec8<T>::V*>(xrow + k);
#pragma unroll
        for (int b = 0; b < RB; ++b)
          if (16 * b + (lane & 15) < p.rank) dv[b] = *reinterpret_cast<const half8*>(drow + static_cast<size_t>(16 * b) * p.K + k);
      }
#pragma unroll
      for (int b = 0; b < RB; ++b) acc[b] = mma16(xv, as_operand(dv[b], T{}), acc[b]);
    }
#pragma unroll
    for (int b = 0; b < RB; ++b) part[wave][b][lane] = acc[b];
    __syncthreads();
    const float sc = p.scale != nullptr ? p.scale[a] : 1.f;
    // lane l of block b holds column 16 b + l % 16 of rows 4 (l / 16) .. + 3
    for (int b = wave; b < RB; b += kWaves) {
      float4v v = part[0][b][lane];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) v += part[w][b][lane];
      const int col = 16 * b + (lane & 15);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 4 * (lane >> 4) + i;
        if (((rows >> r) & 1u) && col < p.rank) p.low[(static_cast<size_t>(split) * p.M + m0 + r) * p.rank + col] = v[i] * sc;
      }
    }
    __syncthreads();
  });
}

// out = y + low @ up^T: a wavefront computes 64 columns of the tile's rows, transposed, so that a lane
// ends up with 16 consecutive columns of one row (rows of block t of the left side: n0 + 16 (i / 4) + 4 t
// + i % 4).
template <bool OUT_F16>
__global__ __launch_bounds__(kThreads) void expand_kernel(Params p) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int slot = blockIdx.x % p.slots, m0 = static_cast<int>(blockIdx.x / p.slots) * kRows;
  const int n0 = (static_cast<int>(blockIdx.y) * kWaves + wave) * 64;
  if (n0 >= p.N) return;
  const int row = m0 + (lane & 15), mine = adapter_of(p, row), q = lane >> 4;
  auto finish = [&](const float4v (&acc)[4]) {
    const size_t at = static_cast<size_t>(row) * p.N + n0 + 16 * q;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (n0 + 16 * q + 8 * h >= p.N) break;
      const float4v a = acc[2 * h] + *reinterpret_cast<const float4v*>(p.y + at + 8 * h);
      const float4v b = acc[2 * h + 1] + *reinterpret_cast<const float4v*>(p.y + at + 8 * h + 4);
      if constexpr (OUT_F16) {
        const float8v v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        *reinterpret_cast<half8*>(static_cast<_Float16*>(p.out) + at + 8 * h) = __builtin_convertvector(v, half8);
      } else {
        *reinterpret_cast<float4v*>(static_cast<float*>(p.out) + at + 8 * h) = a;
        *reinterpret_cast<float4v*>(static_cast<float*>(p.out) + at + 8 * h + 4) = b;
      }
    }
  };
  // rows without an adapter: y as it is (where it is the output already, they are done)
  if (slot == 0 && row < p.M && mine < 0 && p.y != p.out) {
    const float4v none[4] = {};
    finish(none);
  }
  each_adapter(mine, slot, p.slots, [&](int a, uint32_t) {
    const bool ours = mine == a;
    float4v acc[4] = {};
    for (int r0 = 0; r0 < p.rank; r0 += 32) {
      const int r = r0 + 8 * q;
      float8v low = {};
      if (ours && r < p.rank) {
        for (int s = 0; s < p.splits; ++s)
          low += *reinterpret_cast<const float8v*>(p.low + (static_cast<size_t>(s) * p.M + row) * p.rank + r);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int n = n0 + 16 * ((lane & 15) >> 2) + 4 * t + (lane & 3);
        half8 u = {};
        if (n < p.N && r < p.rank) u = *reinterpret_cast<const half8*>(p.up + (static_cast<size_t>(a) * p.N + n) * p.rank + r);
        acc[t] = mma16(widen(u), low, acc[t]);
      }
    }
    if (ours) finish(acc);
  });
}

// ---- host ------------------------------------------------------------------------------------------------

int check(const g16_lora_args& a) {
  if ((a.x_is_f32 | a.out_is_f16) & ~1) return G16_E_DTYPE;
  if (a.M < 0 || a.K < 0 || a.N < 0 || a.adapters < 0 || a.rank < 0 || a.K % 8 != 0 || a.N % 8 != 0 || a.rank % 8 != 0 ||
      a.rank > G16_LORA_MAX_RANK)
    return G16_E_SHAPE;
  if (a.M == 0 || a.N == 0) return G16_OK;
  if (a.x == nullptr || a.down == nullptr || a.up == nullptr || a.index == nullptr || a.y == nullptr || a.out == nullptr) return G16_E_NULL;
  if (!aligned16(a.x) || !aligned16(a.down) || !aligned16(a.up) || !aligned16(a.y) || !aligned16(a.out)) return G16_E_ALIGN;
  return G16_OK;
}

struct Plan {
  int tiles, slots, splits;
};
Plan plan_of(const g16_lora_args& a) {
  const int cus = a.num_cus > 0 ? a.num_cus : 256;
  Plan p;
  p.tiles = ceil_div(a.M, kRows);
  // few tiles: an adapter a workgroup (a tile has at most 16), and K split so that about two land on a CU
  p.slots = p.tiles >= cus ? 1 : (p.tiles * 4 >= cus ? 4 : 16);
  if (p.slots > a.M) p.slots = a.M;
  const int steps = ceil_div(a.K, 32);
  const int want = (2 * cus + p.tiles * p.slots - 1) / (p.tiles * p.slots);
  p.splits = want < 1 ? 1 : (want > 8 ? 8 : want);
  if (p.splits > (steps + 7) / 8) p.splits = (steps + 7) / 8;
  if (p.splits < 1) p.splits = 1;
  return p;
}

Params params(const g16_lora_args& a, const Plan& plan) {
  return Params{a.x, reinterpret_cast<const _Float16*>(a.down), reinterpret_cast<const _Float16*>(a.up), a.index, a.scale, a.y, a.out,
                static_cast<float*>(a.workspace), a.M, a.K, a.N, a.rank, a.adapters, plan.slots, plan.splits};
}

template <typename T>
int run_shrink(const Params& p, const Plan& plan, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(plan.tiles) * plan.slots, plan.splits), block(kThreads);
  if (p.rank <= 16) return launch(shrink_kernel<T, 1>, grid, block, s, p);
  if (p.rank <= 32) return launch(shrink_kernel<T, 2>, grid, block, s, p);
  if (p.rank <= 64) return launch(shrink_kernel<T, 4>, grid, block, s, p);
  return launch(shrink_kernel<T, 8>, grid, block, s, p);
}

}  // namespace
}  // namespace g16

using namespace g16;

extern "C" size_t g16_lora_workspace_bytes(const g16_lora_args* args) {
  if (args == nullptr || check(*args) != G16_OK || args->M == 0 || args->N == 0) return 0;
  return static_cast<size_t>(plan_of(*args).splits) * args->M * args->rank * sizeof(float);
}

extern "C" int g16_lora_shrink(const g16_lora_args* args, void* stream) {
  if (args == nullptr) return G16_E_NULL;
  const int st = check(*args);
  if (st != G16_OK || args->M == 0 || args->N == 0 || args->rank == 0 || args->adapters == 0) return st;
  if (args->workspace == nullptr || static_cast<size_t>(args->workspace_bytes) < g16_lora_workspace_bytes(args)) return G16_E_WORKSPACE;
  if (!aligned16(args->workspace)) return G16_E_ALIGN;
  const Plan plan = plan_of(*args);
  const Params p = params(*args, plan);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return args->x_is_f32 ? run_shrink<float>(p, plan, s) : run_shrink<_Float16>(p, plan, s);
}

extern "C" int g16_lora_expand(const g16_lora_args* args, void* stream) {
  if (args == nullptr) return G16_E_NULL;
  const int st = check(*args);
  if (st != G16_OK || args->M == 0 || args->N == 0) return st;
  if (args->rank > 0 && args->adapters > 0 &&
      (args->workspace == nullptr || static_cast<size_t>(args->workspace_bytes) < g16_lora_workspace_bytes(args)))
    return G16_E_WORKSPACE;
  if (!aligned16(args->workspace)) return G16_E_ALIGN;
  const Plan plan = plan_of(*args);
  const Params p = params(*args, plan);
  const dim3 grid(static_cast<unsigned>(plan.tiles) * plan.slots, (args->N + 64 * kWaves - 1) / (64 * kWaves)), block(kThreads);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return args->out_is_f16 ? launch(expand_kernel<true>, grid, block, s, p) : launch(expand_kernel<false>, grid, block, s, p);
}
