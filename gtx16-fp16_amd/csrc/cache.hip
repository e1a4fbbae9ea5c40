// A cache of keys and values in 8 bits: written as tokens arrive (g16_cache_write) and read back as rows
// (g16_cache_read). The formats stand in g16.h.
//
// Both pass over their data once and are bound by memory. A run is the d values of one token's head; LP lanes have it, 8
// values each, and find its largest magnitude by exchanges within a row of 16 lanes.
#include <type_traits>

#include "code8.hpp"

namespace g16 {
namespace {

constexpr int kThreads = 256;

// Keys or values: workgroups are told apart by blockIdx.y, so that what is here stays in scalar registers.
struct Side {
  char* rows;
  uint8_t* codes;
  float* scales;
  int64_t token, head;                                       // bytes, of the rows
  int64_t c_page, c_token, c_head, s_page, s_token, s_head;  // elements: bytes of the codes
};
struct Params {
  Side side[2];
  const int32_t* slots;
  Divide page, hkv, block;  // by a page's tokens; by the heads; to read: by block_rows where runs go row by row within a head, else by 1
  uint32_t n, d, capacity;  // capacity: slots
  uint32_t block_rows;
};

// The largest of LP lanes' values.
template <int LP>
__device__ inline uint32_t largest(uint32_t v) {
  auto with = [&](auto ctrl) {
    v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), decltype(ctrl)::value, 0xf, 0xf, true)));
  };
  if constexpr (LP >= 2) with(std::integral_constant<int, 0xb1>{});    // lane ^ 1
  if constexpr (LP >= 4) with(std::integral_constant<int, 0x4e>{});    // lane ^ 2
  if constexpr (LP >= 8) with(std::integral_constant<int, 0x141>{});   // 7 - lane, of 8
  if constexpr (LP >= 16) with(std::integral_constant<int, 0x140>{});  // 15 - lane, of 16
  return v;
}

template <typename T>
struct alignas(16) Eight {
  T v[8];
};

// The largest magnitude's bits, as a float's, of eight values. Bits in place of values: NaN is above infinity then, so
// nothing that is not finite is passed over.
__device__ inline uint32_t top_of(const Eight<float>& x) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(x.v[j]) & 0x7fffffffu);
  return m;
}
typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));
__device__ inline uint32_t top_of(const Eight<_Float16>& x) {
  const u32x4 w = __builtin_bit_cast(u32x4, x);
  ushort2v m = {0, 0};
#pragma unroll
  for (int j = 0; j < 4; ++j) m = __builtin_elementwise_max(m, __builtin_bit_cast(ushort2v, w[j] & 0x7fff7fffu));
  const unsigned short h = max(m[0], m[1]);
  return __float_as_uint(static_cast<float>(__builtin_bit_cast(_Float16, h)));
}

// A workgroup: block_rows rows, all heads of them. Of rows with one slot the last is written, so every workgroup looks
// through the later rows' slots, n^2 / block_rows looks in all: a map of its own slots' last bits passes over nearly all of the
// others, and the lanes together, a row each, compare one that it does not, of the same slot in 64 rows only the last. A
// wavefront whose rows have all been found looks no further. (32768 rows of 8 heads of 128, fp16, the same ones again and again:
// 210 us where every lane compared its own with all rows, 46.5 so, 58 for other rows every time; all of one slot: 23 us, where
// each was compared 756.) A launch has at most kLaunchRows: the next one's rows are later ones anyway (2^20 rows of one
// head of 64: 0.90 ms, 1.01 by 16384).
constexpr uint32_t kMapBits = 32 * kThreads, kMostRows = 32, kLaunchRows = 32768;

template <typename T, int CODE, int LP>
__global__ __launch_bounds__(kThreads) void write_kernel(Params p) {
  __shared__ uint32_t slot_of[kMostRows], live[kMostRows], map[kThreads];
  const Side& side = p.side[blockIdx.y];
  const uint32_t tid = threadIdx.x, first = blockIdx.x * p.block_rows, here = min(p.block_rows, p.n - first);
  const uint32_t lane = tid % LP, runs = here * p.hkv.by;
  const bool inside = lane * 8 < p.d;
  Eight<T> x = {};
  auto load = [&](uint32_t run) {
    const uint32_t r = p.hkv(run), h = run - r * p.hkv.by;
    if (run < runs && inside) x = *reinterpret_cast<const Eight<T>*>(side.rows + (first + r) * side.token + h * side.head + lane * 8 * sizeof(T));
  };
  uint32_t run = tid / LP;
  load(run);
  if (tid < here) {
    const uint32_t s = static_cast<uint32_t>(p.slots[first + tid]);  // (negative ones: past every capacity)
    slot_of[tid] = s;
    live[tid] = s < p.capacity;
  }
  map[tid] = 0;
  __syncthreads();
  if (tid < here && live[tid] != 0) atomicOr(&map[(slot_of[tid] % kMapBits) / 32], 1u << (slot_of[tid] % 32));
  __syncthreads();
  constexpr int kLooks = 8;  // under way together
  const uint32_t row = tid % 64, end = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(tid & ~63u))) + 63;  // (lane 63's row)
  uint32_t own = row < here && live[row] != 0 ? slot_of[row] : ~0u;  // ~0: nothing to look for
  for (uint32_t i0 = first + 1; i0 < p.n && __ballot(own != ~0u) != 0; i0 += kLooks * kThreads) {
    uint32_t s[kLooks];
#pragma unroll
    for (int j = 0; j < kLooks; ++j) s[j] = static_cast<uint32_t>(p.slots[min(i0 + tid + j * kThreads, p.n - 1)]);
#pragma unroll
    for (int j = 0; j < kLooks; ++j) {
      const uint32_t i = i0 + tid + j * kThreads;
      const bool maybe = i < p.n && s[j] < p.capacity && (map[(s[j] % kMapBits) / 32] >> (s[j] % 32) & 1) != 0;
      for (uint64_t hits = __ballot(maybe); hits != 0;) {
        const uint32_t slot = static_cast<uint32_t>(__builtin_amdgcn_readlane(s[j], __builtin_ctzll(hits)));
        const uint64_t same = hits & __ballot(s[j] == slot);
        if (own == slot && first + row < i0 + j * kThreads + end - static_cast<uint32_t>(__builtin_clzll(same))) {
          live[row] = 0;
          own = ~0u;
        }
        hits &= ~same;
      }
    }
  }
  __syncthreads();
  for (; run < runs; run += kThreads / LP) {
    const uint32_t r = p.hkv(run), h = run - r * p.hkv.by;
    const Scaling s = scaling_of<CODE>(__uint_as_float(largest<LP>(top_of(x))));
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_f(x.v[j]);
    const u32x2 codes = encode8<CODE>(v, s);
    load(run + kThreads / LP);
    if (live[r] != 0 && inside) {
      const uint32_t page = p.page(slot_of[r]), at = slot_of[r] - page * p.page.by;
      *reinterpret_cast<u32x2*>(side.codes + page * side.c_page + at * side.c_token + h * side.c_head + lane * 8) = codes;
      if (lane == 0) side.scales[page * side.s_page + at * side.s_token + h * side.s_head] = s.scale;
    }
  }
}

// A workgroup: block_rows rows, all heads of them; a thread: eight values of kRuns runs at a time.
constexpr int kRuns = 4;

template <typename T, int CODE, int LP>
__global__ __launch_bounds__(kThreads) void read_kernel(Params p) {
  constexpr uint32_t kStep = kThreads / LP;
  const Side& side = p.side[blockIdx.y];
  const uint32_t lane = threadIdx.x % LP, first = blockIdx.x * p.block_rows, here = min(p.block_rows, p.n - first);
  const bool by_head = p.block.by > 1;
  const uint32_t runs = (by_head ? p.block_rows : here) * p.hkv.by;
  if (lane * 8 >= p.d) return;
  for (uint32_t run0 = threadIdx.x / LP; run0 < runs; run0 += kRuns * kStep) {
    u32x2 codes[kRuns];
    float scale[kRuns];
    uint32_t row[kRuns], h[kRuns], slot[kRuns];
    bool some[kRuns];
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      const uint32_t run = min(run0 + i * kStep, runs - 1);
      uint32_t r;
      if (by_head) {
        h[i] = p.block(run);
        r = run - h[i] * p.block.by;
      } else {
        r = p.hkv(run);
        h[i] = run - r * p.hkv.by;
      }
      some[i] = r < here && run0 + i * kStep < runs;
      row[i] = first + min(r, here - 1);
      slot[i] = static_cast<uint32_t>(p.slots[row[i]]);  // (negative ones: past every capacity)
    }
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      codes[i] = u32x2{0, 0};
      scale[i] = 0.f;
      if (slot[i] >= p.capacity) continue;
      const uint32_t page = p.page(slot[i]), at = slot[i] - page * p.page.by;
      codes[i] = *reinterpret_cast<const u32x2*>(side.codes + page * side.c_page + at * side.c_token + h[i] * side.c_head + lane * 8);
      scale[i] = side.scales[page * side.s_page + at * side.s_token + h[i] * side.s_head];
    }
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      if (!some[i]) continue;
      float v[8];
      decode8<CODE>(codes[i], v);
      Eight<T> x;
#pragma unroll
      for (int j = 0; j < 8; ++j) x.v[j] = static_cast<T>(v[j] * scale[i]);
      *reinterpret_cast<Eight<T>*>(side.rows + ((static_cast<uint64_t>(row[i]) * p.hkv.by + h[i]) * p.d + lane * 8) * sizeof(T)) = x;
    }
  }
}

template <typename T, int CODE, int LP>
int write(Params p, hipStream_t stream) {
  const uint32_t full = kThreads / LP / p.hkv.by, rows = p.n;
  for (uint32_t done = 0; done < rows; done += p.n) {
    p.n = min(rows - done, kLaunchRows);
    // Rows of a workgroup: enough for every lane, and more where there are many workgroups, which all look through the later rows' slots.
    p.block_rows = min(max(max(full, p.n / 1024), 1u), kMostRows);
    const int rc = launch(write_kernel<T, CODE, LP>, dim3((p.n + p.block_rows - 1) / p.block_rows, 2), dim3(kThreads), stream, p);
    if (rc != 0) return rc;
    for (Side& side : p.side) side.rows += p.n * side.token;
    p.slots += p.n;
  }
  return G16_OK;
}
template <typename T, int CODE, int LP>
int read(Params p, hipStream_t stream) {
  p.block_rows = max(kThreads / LP / p.hkv.by * kRuns, 1u);  // enough for every lane, four times
  // A cache whose memory is ordered by heads is read head by head.
  const bool by_head = p.side[0].c_token < p.side[0].c_head && p.n > 64;
  if (by_head) p.block_rows = max(p.block_rows, 16u);
  p.block = divide_by(by_head ? p.block_rows : 1);
  const uint32_t blocks = (p.n + p.block_rows - 1) / p.block_rows;
  if (blocks > (1u << 23) - 1) return G16_E_SHAPE;  // (2^32 threads a launch)
  return launch(read_kernel<T, CODE, LP>, dim3(blocks, 2), dim3(kThreads), stream, p);
}
template <typename T, int CODE, int LP>
int run(const Params& p, bool to_cache, hipStream_t stream) {
  return to_cache ? write<T, CODE, LP>(p, stream) : read<T, CODE, LP>(p, stream);
}
template <typename T, int CODE>
int run(const Params& p, bool to_cache, hipStream_t stream) {
  return p.d <= 8 ? run<T, CODE, 1>(p, to_cache, stream) : p.d <= 16 ? run<T, CODE, 2>(p, to_cache, stream) : p.d <= 32 ? run<T, CODE, 4>(p, to_cache, stream)
         : p.d <= 64 ? run<T, CODE, 8>(p, to_cache, stream) : run<T, CODE, 16>(p, to_cache, stream);
}

// (what the Python binding packs)
static_assert(sizeof(g16_cache_args) == 7 * 8 + 16 * 8 + 8 * 4, "no padding");

int cache(const g16_cache_args* args, bool to_cache, void* stream) {
  if (args == nullptr) return G16_E_NULL;
  const g16_cache_args& a = *args;
  if ((a.is_f32 != 0 && a.is_f32 != 1) || (a.code != G16_CODE_INT8 && a.code != G16_CODE_E4M3)) return G16_E_DTYPE;
  if (a.rows < 0 || a.pages < 0 || a.page < 0 || a.hkv < 0 || a.hkv > (1 << 20) || a.d <= 0 || a.d % 8 != 0 || a.d > G16_ATTENTION_MAX_D) return G16_E_SHAPE;
  if (static_cast<int64_t>(a.pages) * a.page > (1LL << 31) - 1) return G16_E_SHAPE;
  if (a.rows == 0 || a.hkv == 0) return G16_OK;
  const int64_t size = a.is_f32 ? 4 : 2;
  if (a.k == nullptr || a.v == nullptr || a.slots == nullptr) return G16_E_NULL;
  if (!aligned16(a.k) || !aligned16(a.v)) return G16_E_ALIGN;
  const int64_t capacity = static_cast<int64_t>(a.pages) * a.page;
  if (capacity > 0) {
    if (a.k_cache == nullptr || a.v_cache == nullptr || a.k_scale == nullptr || a.v_scale == nullptr) return G16_E_NULL;
    const int64_t all = a.kc_page | a.kc_token | a.kc_head | a.vc_page | a.vc_token | a.vc_head | static_cast<int64_t>(reinterpret_cast<uintptr_t>(a.k_cache)) |
                        static_cast<int64_t>(reinterpret_cast<uintptr_t>(a.v_cache));
    if (all % 8 != 0) return G16_E_ALIGN;
  }
  if (to_cache && (a.k_token * size % 16 != 0 || a.k_head * size % 16 != 0 || a.v_token * size % 16 != 0 || a.v_head * size % 16 != 0)) return G16_E_ALIGN;
  Params p = {};
  p.side[0] = {static_cast<char*>(a.k), static_cast<uint8_t*>(a.k_cache), a.k_scale, a.k_token * size, a.k_head * size,
               a.kc_page, a.kc_token, a.kc_head, a.ks_page, a.ks_token, a.ks_head};
  p.side[1] = {static_cast<char*>(a.v), static_cast<uint8_t*>(a.v_cache), a.v_scale, a.v_token * size, a.v_head * size,
               a.vc_page, a.vc_token, a.vc_head, a.vs_page, a.vs_token, a.vs_head};
  p.slots = a.slots;
  p.n = static_cast<uint32_t>(a.rows);
  p.page = divide_by(static_cast<uint32_t>(a.page > 0 ? a.page : 1));
  p.hkv = divide_by(static_cast<uint32_t>(a.hkv));
  p.d = static_cast<uint32_t>(a.d);
  p.capacity = static_cast<uint32_t>(capacity);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a.code == G16_CODE_INT8) return a.is_f32 ? run<float, G16_CODE_INT8>(p, to_cache, s) : run<_Float16, G16_CODE_INT8>(p, to_cache, s);
  return a.is_f32 ? run<float, G16_CODE_E4M3>(p, to_cache, s) : run<_Float16, G16_CODE_E4M3>(p, to_cache, s);
}

}  // namespace
}  // namespace g16

extern "C" int g16_cache_write(const g16_cache_args* args, void* stream) { return g16::cache(args, true, stream); }
extern "C" int g16_cache_read(const g16_cache_args* args, void* stream) { return g16::cache(args, false, stream); }
