// Low-rank adapters of many requests beside one linear layer (g16_lora_*; formulas in g16.h):
//   low[m, :] = scale[a] * x[m, :] @ down[a]^T,   out[m, :] = y[m, :] + low[m, :] @ up[a]^T,   a = index[m],
// where y is the shared projection's result.
//
// Both products work on tiles of 16 rows on the 16x16 MFMA blocks, one adapter at a time, for whichever
// rows of the tile have it; the rows of a tile are looked at once (a ballot per adapter among them), so
// they may come in any order and need no sorting. The work of a workgroup is dealt to its 8 wavefronts by
// what the tile turns out to hold: one adapter, and they share its K or its columns; 16, and each takes two.
// (Workgroups for adapters that a tile may have cost more than they gave: 2048 of them with nothing to do
// took 10 us.)
//   * shrink, few rows: operands straight from memory, as the adapters (rank * (K + N) * 2 bytes for nearly every
//     row of a decode batch) are what there is to read. K is split over workgroups as well; expand adds the
//     parts up.
//   * shrink, many rows: x and `down` come by DMA into LDS. A fragment straight from memory is 16 rows of 64
//     bytes, whose lanes come in fours of different rows: 64 pieces, and the address unit takes them one by
//     one (4096 x 4096 fp16, rank 32: 22 us).
//   * expand: low is fp32, far from fp16's range in rows of massive activations. A row is scaled by a power of
//     two to 2^14 .. 2^15 and taken as three fp16 parts, each kept 2^11 above its size: all 24 bits of every value
//     down to 2^-38 of the row's largest, past which it adds nothing that fp32 sums keep (`up` is fp16, so columns
//     differ by 2^40 at most). Three 16x16x32 MFMAs, with a sum for each part, replace eight fp32 ones of twice the
//     cycles each. The result passes through LDS, so that y is read and the output written in whole rows of 64 columns.
//   * few rows whose adapters are small: expand computes low itself, in every workgroup (one launch less).
// fp32 activations run on v_mfma_f32_16x16x4_f32: nothing is rounded.
#include "g16_common.hpp"

namespace g16 {
namespace {

typedef float float8v __attribute__((ext_vector_type(8)));

constexpr int kRows = 16;  // rows of a tile
// weights of `down` (rows * rank * K) up to which every workgroup of expand computes low itself
constexpr int64_t kFusedWeights = 1 << 16;
constexpr int kStagedTiles = 16;  // tiles from which shrink takes its operands through LDS
constexpr int kThreads = 512, kWaves = 8;

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
  int M, K, N, rank, adapters, tiles, slots, splits, chunks;
  int first;  // row of the launch's first tile
};

// A row's adapter: -1 for every index that names none.
__device__ inline int adapter_of(const Params& p, int row) {
  const int a = row < p.M ? p.index[row] : -1;
  return a >= 0 && a < p.adapters ? a : -1;
}

// The adapters among a tile's 16 rows. mine: that of row lane % 16 (-1: none); ids: lane i, the i-th.
struct Adapters {
  int mine, count, ids;
  float scale;  // of `mine`
};
__device__ inline Adapters adapters_of(const Params& p, int m0) {
  const int lane = threadIdx.x & 63, row = m0 + (lane & 15);
  Adapters t;
  t.mine = adapter_of(p, row);
  t.scale = t.mine >= 0 && p.scale != nullptr ? p.scale[t.mine] : 1.f;
  t.ids = -1;
  t.count = 0;
  for (uint32_t left = static_cast<uint32_t>(__ballot(t.mine >= 0)) & 0xffffu; left != 0; ++t.count) {
    const int a = __builtin_amdgcn_readlane(t.mine, __builtin_ctz(left));
    left &= ~static_cast<uint32_t>(__ballot(t.mine == a));
    if (lane == t.count) t.ids = a;
  }
  return t;
}

// Steps s0 .. s1 - 1 of 32 values of K of low for the tile's rows and every `groups`-th adapter from `group` on:
// block b of 16 rank columns, lane l: column 16 b + l % 16 of rows 4 (l / 16) .. + 3; other adapters' rows
// stay as they are.
template <typename T, int RB>
__device__ inline void shrink_steps(const Params& p, int m0, const Adapters& t, int group, int groups, int s0, int s1, float4v (&low)[RB]) {
  using V8 = typename Vec8<T>::V;
  const int lane = threadIdx.x & 63, kl = (lane >> 4) * 8;
  const T* xrow = static_cast<const T*>(p.x) + static_cast<size_t>(min(m0 + (lane & 15), p.M - 1)) * p.K;
  for (int i = group; i < t.count; i += groups) {
    const int a = __builtin_amdgcn_readlane(t.ids, i);
    const uint32_t rows = static_cast<uint32_t>(__ballot(t.mine == a));
    const _Float16* drow[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) drow[b] = p.down + (static_cast<size_t>(a) * p.rank + min(16 * b + (lane & 15), p.rank - 1)) * p.K;
    float4v acc[RB] = {};
    // kG steps' loads at a time. They are unconditional, from clamped places: past the share or past K, x counts
    // as zeros (and `down` as values of the same row, which reach no other sum); columns past the rank are
    // not stored.
    constexpr int kG = RB == 1 ? 8 : (RB == 2 ? 4 : 2);
    for (int s = s0; s < s1; s += kG) {
      V8 xv[kG];
      half8 dv[kG][RB];
#pragma unroll
      for (int g = 0; g < kG; ++g) {
        const int k = min(s + g, s1 - 1) * 32 + kl, at = min(k, p.K - 8);
        xv[g] = *reinterpret_cast<const V8*>(xrow + at);
#pragma unroll
        for (int b = 0; b < RB; ++b) dv[g][b] = *reinterpret_cast<const half8*>(drow[b] + at);
        if (s + g >= s1 || k >= p.K) xv[g] = V8{};
      }
#pragma unroll
      for (int g = 0; g < kG; ++g)
#pragma unroll
        for (int b = 0; b < RB; ++b) acc[b] = mma16(xv[g], as_operand(dv[g][b], T{}), acc[b]);
    }
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if ((rows >> (4 * (lane >> 4) + j)) & 1u) low[b][j] = acc[b][j];
  }
}

// The wavefronts' sums (part, in LDS) added up and stored for split `split`, for the rows of every `slots`-th adapter.
template <int RB>
__device__ inline void store_low(const Params& p, int m0, const Adapters& t, int slot, int slots, int split, const float4v (&part)[kWaves][RB][kWave]) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t rows = 0;
  for (int i = slot; i < t.count; i += slots) rows |= static_cast<uint32_t>(__ballot(t.mine == __builtin_amdgcn_readlane(t.ids, i)));
  for (int b = wave; b < RB; b += kWaves) {
    float4v v = part[0][b][lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += part[w][b][lane];
    const int col = 16 * b + (lane & 15);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * (lane >> 4) + i;
      const float sc = __shfl(t.scale, r);
      if (((rows >> r) & 1u) && col < p.rank) p.low[(static_cast<size_t>(split) * p.M + m0 + r) * p.rank + col] = v[i] * sc;
    }
  }
}

// How 8 wavefronts share `count` adapters and a range of K: groups of wavefronts on different adapters, those
// of a group on different parts of K.
__device__ inline int groups_for(int count) { return count >= 5 ? 8 : (count >= 3 ? 4 : (count == 2 ? 2 : 1)); }

// low from memory: a tile's every `slots`-th adapter (workgroups of one tile are `tiles` apart: neighbours go to
// different XCDs), split blockIdx.y of K.
template <typename T, int RB>
__global__ __launch_bounds__(kThreads) void shrink_kernel(Params p) {
  __shared__ float4v part[kWaves][RB][kWave];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m0 = p.first + static_cast<int>(blockIdx.x % p.tiles) * kRows, slot = blockIdx.x / p.tiles, split = blockIdx.y;
  const Adapters t = adapters_of(p, m0);
  if (slot >= t.count) return;
  const int steps = ceil_div(p.K, 32), of = p.splits * kWaves, at = split * kWaves + wave;
  float4v low[RB] = {};
  shrink_steps<T, RB>(p, m0, t, slot, p.slots, static_cast<int>(static_cast<int64_t>(steps) * at / of),
                      static_cast<int>(static_cast<int64_t>(steps) * (at + 1) / of), low);
#pragma unroll
  for (int b = 0; b < RB; ++b) part[wave][b][lane] = low[b];
  __syncthreads();
  store_low<RB>(p, m0, t, slot, p.slots, split, part);
}

// low by way of LDS: kChunk values of K at a time, of x's 16 rows and an adapter's 16 RB rows of `down`, a
// wavefront on 32 of them; the next chunks on their way meanwhile. 16-byte piece c of row r at c ^ r % 16. All
// adapters of a chunk in turn, so that x is read once (1024 x 4096, rank 16, 32 adapters at random: 24.8 us an
// adapter at a time, 23.1 so: 142 MB, mostly of `down`, out of L2 and the Infinity Cache, which twice as many
// steps in flight slowed down to 27).
constexpr int kChunk = 32 * kWaves;
template <typename T, int RB>
struct Stage {
  static constexpr int XROW = kChunk * sizeof(T), DROW = kChunk * 2;  // bytes
  static constexpr int BYTES = 16 * XROW + 16 * RB * DROW;
  static constexpr int XI = 16 * XROW / 1024 / kWaves, DI = 16 * RB * DROW / 1024 / kWaves;  // DMA instructions of a wavefront
  static constexpr int COUNT = 3 * BYTES <= 80 * 1024 ? 3 : 2;
};
template <typename T, int RB>
__global__ __launch_bounds__(kThreads) void shrink_tiles_kernel(Params p) {
  using S = Stage<T, RB>;
  constexpr int kLds = S::COUNT * S::BYTES > kWaves * RB * kWave * 16 ? S::COUNT * S::BYTES : kWaves * RB * kWave * 16;
  __shared__ __attribute__((aligned(1024))) char lds[kLds];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lin = static_cast<int>(blockIdx.x), m0 = p.first + lin % p.tiles * kRows, slot = lin / p.tiles, split = blockIdx.y;
  const Adapters t = adapters_of(p, m0);
  if (slot >= t.count) return;
  const int count = (t.count - slot + p.slots - 1) / p.slots;  // this slot's adapters: slot, slot + slots, ..
  const int all = ceil_div(p.K, kChunk), c0 = static_cast<int>(static_cast<int64_t>(all) * split / p.splits),
            c1 = static_cast<int>(static_cast<int64_t>(all) * (split + 1) / p.splits);
  const uint32_t base = lds_base(lds);
  constexpr int XC = S::XROW / 16, DC = S::DROW / 16;  // pieces of a row
  // Where this lane's pieces of a chunk are, in its rows (`in`: at which value of K).
  uint32_t x_off[S::XI], d_off[S::DI];
  int x_in[S::XI], d_in[S::DI];
#pragma unroll
  for (int n = 0; n < S::XI; ++n) {
    const int row = (wave * S::XI + n) * (64 / XC) + lane / XC, c = (lane % XC) ^ (row & 15);
    x_in[n] = c * static_cast<int>(16 / sizeof(T));
    x_off[n] = m0 + row < p.M ? static_cast<uint32_t>(row) * p.K * static_cast<uint32_t>(sizeof(T)) + c * 16 : kOob;
  }
#pragma unroll
  for (int n = 0; n < S::DI; ++n) {
    const int row = (wave * S::DI + n) * (64 / DC) + lane / DC, c = (lane % DC) ^ (row & 15);
    d_in[n] = c * 8;
    d_off[n] = row < p.rank ? static_cast<uint32_t>(row) * p.K * 2u + c * 16 : kOob;
  }
  // step `it`: chunk it / count for the slot's adapter it % count, x with the chunk's first
  int chunk = c0, which = 0, to = 0;  // of the next step to load, and its place
  const size_t adapter = static_cast<size_t>(p.rank) * p.K;
  auto issue = [&]() {
    const int k0 = chunk * kChunk, left = p.K - k0;
    const uint32_t at = base + to * S::BYTES + wave * (S::XI * 1024);
    if (which == 0) {
      const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<T*>(static_cast<const T*>(p.x) + static_cast<size_t>(m0) * p.K + k0), 0, 0x7fffffff, kRawBufferDword3);
#pragma unroll
      for (int n = 0; n < S::XI; ++n) dma16(rx, at + n * 1024, x_in[n] < left ? x_off[n] : kOob);
    }
    const int a = __builtin_amdgcn_readlane(t.ids, slot + which * p.slots);
    const __amdgpu_buffer_rsrc_t rd =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<_Float16*>(p.down + a * adapter + k0), 0, 0x7fffffff, kRawBufferDword3);
#pragma unroll
    for (int n = 0; n < S::DI; ++n)
      dma16(rd, base + to * S::BYTES + 16 * S::XROW + (wave * S::DI + n) * 1024, d_in[n] < left ? d_off[n] : kOob);
    to = to + 1 == S::COUNT ? 0 : to + 1;
    if (++which == count) {
      which = 0;
      ++chunk;
    }
  };
  const int total = count * (c1 - c0), r16 = lane & 15, q = lane >> 4;
  for (int i = 0; i < S::COUNT - 1; ++i)
    if (i < total) issue();
  int row_of[4];  // the adapters of rows 4 q .. 4 q + 3
#pragma unroll
  for (int j = 0; j < 4; ++j) row_of[j] = __shfl(t.mine, 4 * q + j);
  float4v low[RB] = {};
  typename Vec8<T>::V xv = {};
  const char* at = lds;
  for (int it = 0, now = 0; it < total; ++it, now = now + 1 == count ? 0 : now + 1) {
    // step `it` has arrived: only the younger ones may be in flight (one with x in it is XI instructions longer)
    if (S::COUNT == 3 && it + 1 < total) {
      if (now + 1 == count) wait_dma_le<S::XI + S::DI>();
      else wait_dma_le<S::DI>();
    } else {
      wait_dma_le<0>();
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    phase_barrier();  // ... for every wavefront, and every one has read the step whose place the next one takes
    if (it + S::COUNT - 1 < total) issue();
    if (now == 0) {
      if constexpr (sizeof(T) == 2) {
        xv = *reinterpret_cast<const half8*>(at + r16 * S::XROW + (((wave * 4 + q) ^ r16) << 4));
      } else {
        const float4v a = *reinterpret_cast<const float4v*>(at + r16 * S::XROW + (((wave * 8 + 2 * q) ^ r16) << 4));
        const float4v b = *reinterpret_cast<const float4v*>(at + r16 * S::XROW + (((wave * 8 + 2 * q + 1) ^ r16) << 4));
        xv = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
      }
    }
    // the adapter's rows take the new sums, the others keep theirs
    const int a = __builtin_amdgcn_readlane(t.ids, slot + now * p.slots);
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      const half8 dv = *reinterpret_cast<const half8*>(at + 16 * S::XROW + (16 * b + r16) * S::DROW + (((wave * 4 + q) ^ r16) << 4));
      const float4v sum = mma16(xv, as_operand(dv, T{}), low[b]);
#pragma unroll
      for (int j = 0; j < 4; ++j) low[b][j] = row_of[j] == a ? sum[j] : low[b][j];
    }
    at = at == lds + (S::COUNT - 1) * S::BYTES ? lds : at + S::BYTES;
  }
  __syncthreads();
  auto& part = *reinterpret_cast<float4v(*)[kWaves][RB][kWave]>(lds);
#pragma unroll
  for (int b = 0; b < RB; ++b) part[wave][b][lane] = low[b];
  __syncthreads();
  store_low<RB>(p, m0, t, slot, p.slots, split, part);
}

// out = y + low @ up^T for 64 rows and p.chunks runs of 64 columns from blockIdx.y on. The wavefronts, and the
// gridDim.z workgroups of the same rows and columns, share all (adapter, run) pairs; a pair's part of `up` is
// loaded once for its rows (its fragments are 64 pieces a load, like shrink's: with 16 rows a workgroup they
// took more time than y and the output, 4096 x 4096, rank 64: 47 us). The rows' low is summed up and
// scaled once, into LDS. Bound by y and the output: 4111 x 4096, rank 32, fp16, is 101 MB in 25 us, 4 TB/s.
// RC: pieces of 32 rank columns.
constexpr int kScrRow = 68;   // floats of a row of the wavefronts' LDS: rows start 4 banks apart
constexpr int kManyRows = 64;
template <bool OUT_F16>
__device__ inline void store4(const Params& p, size_t at, float4v v) {
  if constexpr (OUT_F16) *reinterpret_cast<half4*>(static_cast<_Float16*>(p.out) + at) = __builtin_convertvector(v, half4);
  else *reinterpret_cast<float4v*>(static_cast<float*>(p.out) + at) = v;
}
// 2^e that takes `top`, a row's largest value, to 2^14 .. 2^15 (e held to what fp32 has both ways; 0 for infinities)
__device__ inline int exponent_for(float top) {
  return top > 0.f && top < __builtin_huge_valf() ? min(max(14 - ilogbf(top), -120), 120) : 0;
}
// A value of a row with infinities: what is finite in it changes nothing, and might not fit fp16.
__device__ inline float beside_infinity(float v) { return fabsf(v) < __builtin_huge_valf() ? 0.f : v; }

// v = hi + 2^-11 (mid + 2^-11 lo). odd: rows with infinities, which have one part.
struct Parts {
  half8 hi, mid, lo;
};
__device__ inline Parts parts_of(float8v v, bool odd) {
  Parts p;
  p.hi = __builtin_convertvector(v, half8);
  v = (v - widen(p.hi)) * 0x1p11f;
  p.mid = __builtin_convertvector(v, half8);
  v = (v - widen(p.mid)) * 0x1p11f;
  p.lo = __builtin_convertvector(v, half8);
  if (odd) p.mid = p.lo = half8{};
  return p;
}
// 4 columns of `up` times a row's parts
template <int RC>
__device__ inline float4v mma_parts(const half8 (&up)[RC][4], int b, const Parts (&low)[RC]) {
  float4v hi = {}, mid = {}, lo = {};
#pragma unroll
  for (int c = 0; c < RC; ++c) {
    hi = mma16(up[c][b], low[c].hi, hi);
    mid = mma16(up[c][b], low[c].mid, mid);
    lo = mma16(up[c][b], low[c].lo, lo);
  }
  return hi + 0x1p-11f * (mid + 0x1p-11f * lo);
}
template <bool OUT_F16, int RC>
__global__ __launch_bounds__(kThreads, RC == 1 ? 4 : 2) void expand_kernel(Params p) {
  constexpr int kLow = 32 * RC + 4;  // floats of a row: rows start 4 banks times an odd number apart
  __shared__ __attribute__((aligned(16))) float s_low[kManyRows][kLow];
  __shared__ float s_back[kManyRows];  // negative: a row with infinities
  __shared__ __attribute__((aligned(16))) float scratch[kWaves][kRows][kScrRow];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m0 = p.first + static_cast<int>(blockIdx.x) * kManyRows, q = lane >> 4;
  // the adapter of row m0 + lane, and the list of all
  const int mine = adapter_of(p, m0 + lane);
  int ids = -1, count = 0;
  for (uint64_t left = __ballot(mine >= 0); left != 0; ++count) {
    const int a = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
    left &= ~__ballot(mine == a);
    if (lane == count) ids = a;
  }
  {
    const int r = tid >> 3, part = tid & 7;  // 8 threads a row
    const bool some = __shfl(mine, r) >= 0;
    float4v v[RC];
    float top = 0.f;
#pragma unroll
    for (int c = 0; c < RC; ++c) {
      const int e = 32 * c + 4 * part;
      v[c] = float4v{0.f, 0.f, 0.f, 0.f};
      if (some && e < p.rank) {
        const float* from = p.low + static_cast<size_t>(m0 + r) * p.rank + e;
        for (int s = 0; s < p.splits; s += 4) {  // (four splits' loads at a time)
          float4v u[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            u[i] = *reinterpret_cast<const float4v*>(from + static_cast<size_t>(min(s + i, p.splits - 1)) * p.M * p.rank);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (s + i < p.splits) v[c] += u[i];
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(v[c][i]));
    }
#pragma unroll
    for (int i = 1; i < 8; i *= 2) top = fmaxf(top, __shfl_xor(top, i));
    const int e = exponent_for(top);
    const float by = ldexpf(1.f, e);
    const bool odd = top == __builtin_huge_valf();
#pragma unroll
    for (int c = 0; c < RC; ++c) {
      float4v x = v[c] * by;
      if (odd) x = float4v{beside_infinity(x[0]), beside_infinity(x[1]), beside_infinity(x[2]), beside_infinity(x[3])};
      *reinterpret_cast<float4v*>(&s_low[r][32 * c + 4 * part]) = x;
    }
    if (part == 0) s_back[r] = odd ? -1.f : ldexpf(1.f, -e);
  }
  __syncthreads();
  // The pairs: rows without an adapter count as one more (number `count`) where y has to be copied.
  const int n_first = static_cast<int>(blockIdx.y) * p.chunks * 64, runs = min(p.chunks, ceil_div(p.N - n_first, 64));
  const bool copy = p.y != p.out && __ballot(mine < 0 && m0 + lane < p.M) != 0;
  const int pairs = (count + (copy ? 1 : 0)) * runs;
  const int waves = kWaves * gridDim.z, w = wave + kWaves * blockIdx.z;
  const int p0 = static_cast<int>(static_cast<int64_t>(pairs) * w / waves), p1 = static_cast<int>(static_cast<int64_t>(pairs) * (w + 1) / waves);
  float(*scr)[kScrRow] = scratch[wave];
  const int col = (lane & 15) * 4;  // y and the output: lane l holds columns col .. + 3 of rows l / 16 + 4 j
  for (int pair = p0; pair < p1; ++pair) {
    const int which = pair / runs, n = n_first + (pair % runs) * 64;
    const int a = which < count ? __builtin_amdgcn_readlane(ids, which) : -1;
    const uint64_t rows = __ballot(mine == a && m0 + lane < p.M);
    half8 up[RC][4];
    if (a >= 0) {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        // (clamped: low is zero past the rank, and columns past the end are not stored)
        const _Float16* from = p.up + (static_cast<size_t>(a) * p.N + min(n + 16 * b + (lane & 15), p.N - 1)) * p.rank;
#pragma unroll
        for (int c = 0; c < RC; ++c) up[c][b] = *reinterpret_cast<const half8*>(from + min(32 * c + 8 * q, p.rank - 8));
      }
    }
    // The pair's rows, in order: lane k holds the k-th one's number (the others' follow), so that rows in no order
    // at all cost a pair one tile of 16 rather than four (2000 x 2048 x 2048, rank 16, 32 adapters at random:
    // 22 us against 38).
    const int here = __popcll(rows);
    const int before = static_cast<int>(__builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(rows >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(rows), 0)));
    const int order = __builtin_amdgcn_ds_permute(4 * (((rows >> lane) & 1u) != 0 ? before : here + lane - before), lane);
    // y and the output by buffer accesses, out of range (no load, no store) for lanes without a row or column:
    // under a branch, the compiler could not tell how many stores are in flight and would wait for all of
    // them wherever it waits for a load.
    const bool inside = n + col < p.N;
    auto base = [&](const void* m, uint32_t size) {
      return __builtin_amdgcn_make_buffer_rsrc(
          const_cast<char*>(static_cast<const char*>(m)) + (static_cast<size_t>(m0) * p.N + n) * size, 0, 0x7fffffff, kRawBufferDword3);
    };
    const __amdgpu_buffer_rsrc_t r_y = base(p.y, 4), r_out = base(p.out, OUT_F16 ? 2 : 4);
    uint32_t at[2][4];  // elements from there on
    float4v y[2][4];
    auto load_y = [&](int s) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = 16 * s + 4 * j + q, r = __shfl(order, k);
        const bool ok = inside && k < here;
        at[s & 1][j] = ok ? static_cast<uint32_t>(r) * static_cast<uint32_t>(p.N) + col : kOob;
        y[s & 1][j] = __builtin_bit_cast(float4v, __builtin_amdgcn_raw_buffer_load_b128(r_y, static_cast<int>(ok ? at[s & 1][j] * 4 : kOob), 0, 0));
      }
    };
    load_y(0);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      float4v(&v)[4] = y[s & 1];
      if (s < 3) load_y(s + 1);
      if (a >= 0) {
        const int r = __shfl(order, 16 * s + (lane & 15));
        const float back = s_back[r];
        Parts low[RC];
#pragma unroll
        for (int c = 0; c < RC; ++c) {
          const float4v x = *reinterpret_cast<const float4v*>(&s_low[r][32 * c + 8 * q]);
          const float4v y = *reinterpret_cast<const float4v*>(&s_low[r][32 * c + 8 * q + 4]);
          low[c] = parts_of(__builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7), back < 0.f);
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          // lane l: columns 16 b + 4 (l / 16) .. + 3 of row l % 16
          *reinterpret_cast<float4v*>(&scr[lane & 15][16 * b + 4 * q]) = mma_parts<RC>(up, b, low) * fabsf(back);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += *reinterpret_cast<const float4v*>(&scr[q + 4 * j][col]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t e = at[s & 1][j];
        if constexpr (OUT_F16)
          __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, __builtin_convertvector(v[j], half4)), r_out, static_cast<int>(e == kOob ? kOob : e * 2), 0, 0);
        else
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v[j]), r_out, static_cast<int>(e == kOob ? kOob : e * 4), 0, 0);
      }
      if (16 * s + 16 >= here) break;
    }
  }
}

// Few rows whose adapters are small (one tile): low is computed here, by every workgroup for its 64 columns.
// T: of x.
template <typename T, bool OUT_F16, int RC>
__global__ __launch_bounds__(kThreads) void fused_kernel(Params p) {
  constexpr int RB = 2 * RC;
  __shared__ float4v part[kWaves][RB][kWave];
  __shared__ __attribute__((aligned(16))) float scratch[kWaves][kRows][kScrRow];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int m0 = blockIdx.x * kRows, q = lane >> 4, row = m0 + (lane & 15);
  const Adapters t = adapters_of(p, m0);
  // The pairs: rows without an adapter count as one more (number t.count) where y has to be copied.
  const int n_first = static_cast<int>(blockIdx.y) * p.chunks * 64, runs = min(p.chunks, ceil_div(p.N - n_first, 64));
  const bool copy = p.y != p.out && __ballot(t.mine < 0 && row < p.M) != 0;
  const int pairs = (t.count + (copy ? 1 : 0)) * runs;
  const int waves = kWaves * gridDim.z, w = wave + kWaves * blockIdx.z, p0 = pairs * w / waves, p1 = pairs * (w + 1) / waves;
  float(*scr)[kScrRow] = scratch[wave];
  Parts parts[RC];
  float back = 1.f;
  int at = -1, a = -1;
  half8 up[RC][4];
  float4v y[4];
  // y and the output: lane l holds columns 4 (l % 16) .. + 3 of rows l / 16 + 4 j
  const int col = (lane & 15) * 4;
  bool ours[4];
  auto load = [&](int pair) {
    const int which = pair / runs, n = n_first + (pair % runs) * 64;
    const int id = which < t.count ? __builtin_amdgcn_readlane(t.ids, which) : -1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = q + 4 * j, of = __shfl(t.mine, r);  // (by every lane)
      ours[j] = of == id && m0 + r < p.M && n + col < p.N;
      if (ours[j]) y[j] = *reinterpret_cast<const float4v*>(p.y + static_cast<size_t>(m0 + r) * p.N + n + col);
    }
    if (id >= 0) {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        // (clamped: low is zero past the rank, and columns past the end are not stored)
        const _Float16* from = p.up + (static_cast<size_t>(id) * p.N + min(n + 16 * b + (lane & 15), p.N - 1)) * p.rank;
#pragma unroll
        for (int c = 0; c < RC; ++c) up[c][b] = *reinterpret_cast<const half8*>(from + min(32 * c + 8 * q, p.rank - 8));
      }
    }
  };
  // this lane's row (lane % 16) of low: 8 values of every piece, of other adapters' rows zeros
  auto load_low = [&]() {
    float8v low[RC];
    float top = 0.f;
#pragma unroll
    for (int c = 0; c < RC; ++c) {
      const int r = 32 * c + 8 * q;
      low[c] = float8v{};
      if (t.mine == a && r < p.rank) {
        const int rr = lane & 15;
#pragma unroll
        for (int i = 0; i < 8; ++i) low[c][i] = part[0][(r + i) >> 4][((r + i) & 15) + 16 * (rr >> 2)][rr & 3] * t.scale;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(low[c][i]));
    }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const int e = exponent_for(top);
    const float by = ldexpf(1.f, e);
    const bool odd = top == __builtin_huge_valf();
    back = ldexpf(1.f, -e);
#pragma unroll
    for (int c = 0; c < RC; ++c) {
      float8v v = low[c] * by;
      if (odd) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = beside_infinity(v[i]);
      }
      parts[c] = parts_of(v, odd);
    }
  };
  if (p0 < p1) load(p0);
  {
    const int steps = ceil_div(p.K, 32), groups = groups_for(t.count), parts = kWaves / groups, at = wave % parts;
    float4v low[RB] = {};
    shrink_steps<T, RB>(p, m0, t, wave / parts, groups, steps * at / parts, steps * (at + 1) / parts, low);
#pragma unroll
    for (int b = 0; b < RB; ++b) part[wave][b][lane] = low[b];
    __syncthreads();
    for (int i = tid; i < RB * kWave; i += kThreads) {
      float4v v = part[0][i / kWave][i % kWave];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) v += part[w][i / kWave][i % kWave];
      part[0][i / kWave][i % kWave] = v;
    }
    __syncthreads();
  }
  for (int pair = p0; pair < p1; ++pair) {
    const int which = pair / runs, n = n_first + (pair % runs) * 64;
    if (which != at) {
      at = which;
      a = which < t.count ? __builtin_amdgcn_readlane(t.ids, which) : -1;
      if (a >= 0) load_low();
    }
    if (a >= 0) {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        // lane l: columns 16 b + 4 (l / 16) .. + 3 of row l % 16
        *reinterpret_cast<float4v*>(&scr[lane & 15][16 * b + 4 * q]) = mma_parts<RC>(up, b, parts) * back;
      }
    }
    float4v v[4];
    bool mine[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = y[j];
      mine[j] = ours[j];
    }
    if (pair + 1 < p1) load(pair + 1);
    if (a >= 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += *reinterpret_cast<const float4v*>(&scr[q + 4 * j][col]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (!mine[j]) continue;
      store4<OUT_F16>(p, static_cast<size_t>(m0 + q + 4 * j) * p.N + n + col, v[j]);
    }
  }
}

// ---- host ------------------------------------------------------------------------------------------------

int check(const g16_lora_args& a) {
  if ((a.x_is_f32 | a.out_is_f16) & ~1) return G16_E_DTYPE;
  if (a.M < 0 || a.M > INT32_MAX - kManyRows || a.K < 0 || a.N < 0 || a.adapters < 0 || a.rank < 0 || a.K % 8 != 0 || a.N % 8 != 0 || a.rank % 8 != 0 ||
      a.rank > G16_LORA_MAX_RANK || a.K > G16_LORA_MAX_SIDE || a.N > G16_LORA_MAX_SIDE)
    return G16_E_SHAPE;
  if (a.M == 0 || a.N == 0) return G16_OK;
  if (a.x == nullptr || a.down == nullptr || a.up == nullptr || a.index == nullptr || a.y == nullptr || a.out == nullptr) return G16_E_NULL;
  if (!aligned16(a.x) || !aligned16(a.down) || !aligned16(a.up) || !aligned16(a.y) || !aligned16(a.out)) return G16_E_ALIGN;
  return G16_OK;
}

struct Plan {
  bool fused, staged;
  int tiles, slots, splits, chunks, wide;  // wide: workgroups that share a tile's columns in expand
};
Plan plan_of(const g16_lora_args& a) {
  const int cus = a.num_cus > 0 ? a.num_cus : 256;
  Plan p;
  p.tiles = ceil_div(a.M, kRows);
  p.fused = a.M <= kRows && static_cast<int64_t>(a.M) * a.rank * a.K <= kFusedWeights;
  p.staged = p.tiles >= kStagedTiles && a.K >= 2 * kChunk;
  // Staged: K in as many parts as make about two workgroups a CU, of at least two chunks; else up to 8 steps of K a
  // wavefront. Few tiles: an adapter a workgroup (a tile has at most 16). More: the adapters a tile may have on as many
  // workgroups as still make two a CU, eight where they read little each (with 16 for every tile, 100000 rows of
  // 256, rank 16, 8 adapters: 499 us in runs 228, so 431 and 165; 4000 rows, 32 at random: 70, with two a CU 75).
  p.splits = p.staged ? (2 * cus + p.tiles - 1) / p.tiles : ceil_div(ceil_div(a.K, 32), 8 * kWaves);
  const int most = p.staged ? (a.K / (2 * kChunk) < 4 ? a.K / (2 * kChunk) : 4) : 8;
  if (p.splits > most) p.splits = most;
  if (p.splits < 1) p.splits = 1;
  p.slots = p.tiles < kStagedTiles ? kRows : static_cast<int>((p.staged ? 2 : 8) * cus / (static_cast<int64_t>(p.tiles) * p.splits));
  if (p.slots > kRows) p.slots = kRows;
  if (p.slots > a.M) p.slots = a.M;
  if (p.slots < 1) p.slots = 1;
  // expand: about two workgroups a CU, of 1 to 32 runs of 64 columns, several for the same rows and columns
  // where that leaves CUs without any; fused: a run each
  const int runs = ceil_div(a.N, 64), many = ceil_div(a.M, kManyRows);
  const int64_t each = (static_cast<int64_t>(many) * runs + 2 * cus - 1) / (2 * cus);
  p.chunks = p.fused || each < 1 ? 1 : (each > 32 ? 32 : static_cast<int>(each));
  const int64_t groups = static_cast<int64_t>(many) * ceil_div(runs, p.chunks);
  p.wide = p.fused || a.M <= kWaves || groups >= cus ? 1 : static_cast<int>(2 * cus / groups);
  if (p.wide > 8) p.wide = 8;
  return p;
}

Params params(const g16_lora_args& a, const Plan& plan) {
  return Params{a.x, reinterpret_cast<const _Float16*>(a.down), reinterpret_cast<const _Float16*>(a.up), a.index, a.scale, a.y, a.out,
                static_cast<float*>(a.workspace), a.M, a.K, a.N, a.rank, a.adapters, plan.tiles, plan.slots, plan.splits, plan.chunks, 0};
}

// A launch's workgroups in x: 2^32 threads, which the rows of the largest batches pass; they are dealt to several.
constexpr int kMostGroups = (1 << 23) - 1;

template <typename T, int RB>
int run_shrink_as(Params p, const Plan& plan, hipStream_t s) {
  const dim3 block(kThreads);
  const int all = plan.tiles, most = kMostGroups / plan.slots;
  int rc = 0;
  for (int t = 0; t < all && rc == 0; t += most) {
    p.tiles = all - t < most ? all - t : most;
    p.first = t * kRows;
    const dim3 grid(p.tiles * plan.slots, plan.splits);
    rc = plan.staged ? launch(shrink_tiles_kernel<T, RB>, grid, block, s, p) : launch(shrink_kernel<T, RB>, grid, block, s, p);
  }
  return rc;
}
template <typename T>
int run_shrink(const Params& p, const Plan& plan, hipStream_t s) {
  if (p.rank <= 16) return run_shrink_as<T, 1>(p, plan, s);
  if (p.rank <= 32) return run_shrink_as<T, 2>(p, plan, s);
  if (p.rank <= 64) return run_shrink_as<T, 4>(p, plan, s);
  return run_shrink_as<T, 8>(p, plan, s);
}

template <bool OUT_F16>
int run_expand(Params p, const Plan& plan, hipStream_t s) {
  const dim3 block(kThreads);
  const int all = ceil_div(p.M, kManyRows);
  int rc = 0;
  for (int t = 0; t < all && rc == 0; t += kMostGroups) {
    p.first = t * kManyRows;
    const dim3 grid(all - t < kMostGroups ? all - t : kMostGroups, ceil_div(ceil_div(p.N, 64), plan.chunks), plan.wide);
    rc = p.rank <= 32   ? launch(expand_kernel<OUT_F16, 1>, grid, block, s, p)
         : p.rank <= 64 ? launch(expand_kernel<OUT_F16, 2>, grid, block, s, p)
                        : launch(expand_kernel<OUT_F16, 4>, grid, block, s, p);
  }
  return rc;
}
template <typename T, bool OUT_F16>
int run_fused(const Params& p, hipStream_t s) {
  const dim3 grid(1, ceil_div(p.N, 64)), block(kThreads);
  if (p.rank <= 32) return launch(fused_kernel<T, OUT_F16, 1>, grid, block, s, p);
  if (p.rank <= 64) return launch(fused_kernel<T, OUT_F16, 2>, grid, block, s, p);
  return launch(fused_kernel<T, OUT_F16, 4>, grid, block, s, p);
}

}  // namespace
}  // namespace g16

using namespace g16;

extern "C" size_t g16_lora_workspace_bytes(const g16_lora_args* args) {
  if (args == nullptr || check(*args) != G16_OK || args->M == 0 || args->N == 0) return 0;
  const Plan plan = plan_of(*args);
  return plan.fused ? 0 : static_cast<size_t>(plan.splits) * args->M * args->rank * sizeof(float);
}

extern "C" int g16_lora_shrink(const g16_lora_args* args, void* stream) {
  if (args == nullptr) return G16_E_NULL;
  const int st = check(*args);
  if (st != G16_OK || args->M == 0 || args->N == 0 || args->rank == 0 || args->adapters == 0) return st;
  if (plan_of(*args).fused) return G16_OK;
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
  if (args->rank == 0 && args->adapters > 0) return G16_E_SHAPE;  // (the kernels clamp to a row's last 8 values)
  const Plan plan = plan_of(*args);
  if (args->adapters > 0 && !plan.fused &&
      (args->workspace == nullptr || static_cast<size_t>(args->workspace_bytes) < g16_lora_workspace_bytes(args)))
    return G16_E_WORKSPACE;
  if (!aligned16(args->workspace)) return G16_E_ALIGN;
  const Params p = params(*args, plan);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (!plan.fused) return args->out_is_f16 ? run_expand<true>(p, plan, s) : run_expand<false>(p, plan, s);
  if (args->x_is_f32) return args->out_is_f16 ? run_fused<float, true>(p, s) : run_fused<float, false>(p, s);
  return args->out_is_f16 ? run_fused<_Float16, true>(p, s) : run_fused<_Float16, false>(p, s);
}
