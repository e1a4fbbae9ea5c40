// Rotary positions by one axis or several (g16_rotary; the formulas stand in g16.h).
//
// The pass reads and writes every value once and is bound by memory. A thread has V pairs of one row, takes their angles once
// and turns the pairs of several of the row's heads by them: an angle costs about 30 instructions, of which eleven in
// 64 bits, a rotated pair four.
#include "g16_common.hpp"

namespace g16 {
namespace {

constexpr int kThreads = 256;

struct Params {
  const char* x;
  char* out;
  const int32_t* positions;
  const float* freqs;
  int64_t x_seq, x_token, x_head;  // bytes
  uint32_t rows, tokens, heads, d, pairs;
  uint32_t ends[G16_ROTARY_MAX_AXES - 1];  // first pair of the second, third, .. axis
  uint32_t items, turned;                  // pieces of a head's values, and how many of them hold pairs
  uint32_t slices;                         // threads that share a row's heads for one piece
};

template <typename T, int N>
struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Run {
  T v[N];
};

// cos and sin of position * freq radians. Quarter turns for each position, freq * 2 / pi, are held as the sum of two doubles, and what the
// position times the first has over a whole number of them is one fma's, without a product rounded before: 2^-54 of a quarter and
// 2^-104 of the angle are lost, whatever the angle (with one double and a rounded product 2^-52 of it: 1e-7 radians from 2^29
// on). Of the whole quarters only the last two bits matter; what is left, at most half of one, goes through polynomials
// fitted to sin(f pi / 2) / f and (cos(f pi / 2) - 1) / f^2 in f^2 by least squares, reweighted to even errors (largest 4e-9 and 7e-11;
// in fp32 1e-7 and 6e-8).
__device__ inline void turn(double position, double freq, float& c, float& s) {
  constexpr double k2OverPi = 0.63661977236758134308, k2OverPiRest = -3.935735335036497e-17;
  const double rate = freq * k2OverPi, rate_rest = fma(freq, k2OverPiRest, fma(freq, k2OverPi, -rate));
  const double magic = 6755399441055744.0;  // 1.5 * 2^52: a sum with it has whole numbers' bits at its end
  const double shifted = fma(position, rate, magic);
  const double left = fma(position, rate_rest, fma(position, rate, -(shifted - magic)));
  const double more = __builtin_rint(left);  // (the second double's part may add to a half: an eighth at 2^51)
  const uint32_t q = static_cast<uint32_t>(__double_as_longlong(shifted)) + static_cast<uint32_t>(static_cast<int>(more));
  const float f = static_cast<float>(left - more), u = f * f;
  float a = fmaf(u, -0.00460165785625577f, 0.07968003302812576f);
  a = fmaf(u, a, -0.6459634900093079f);
  a = fmaf(u, a, 1.5707963705062866f) * f;
  float b = fmaf(u, 0.0009037665440700948f, -0.02086016535758972f);
  b = fmaf(u, b, 0.25366923213005066f);
  b = fmaf(u, b, -1.2337005138397217f);
  b = fmaf(u, b, 1.f);
  c = (q & 1) ? a : b;
  s = (q & 1) ? b : a;
  c = ((q + 1) & 2) ? -c : c;
  s = (q & 2) ? -s : s;
}

// A thread: piece blockIdx.x * kThreads + threadIdx.x of [row][slice][piece of a head]. The first `turned` pieces of a head are V
// pairs each, the others W values that are copied.
template <typename T, int V, bool NEIGHBOURS>
__global__ __launch_bounds__(kThreads) void rotary_kernel(Params p) {
  constexpr int W = 2 * V < 8 ? 2 * V : 8;
  constexpr int kAhead = 4;  // heads whose loads are under way together
  const uint64_t id = static_cast<uint64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const uint32_t per = p.items * p.slices;
  const uint32_t row = static_cast<uint32_t>(id / per), rest = static_cast<uint32_t>(id % per);
  if (row >= p.rows) return;
  const uint32_t slice = rest / p.items, item = rest % p.items;
  const uint32_t seq = row / p.tokens;
  const char* x = p.x + seq * p.x_seq + (row - seq * p.tokens) * p.x_token;
  char* out = p.out + static_cast<uint64_t>(row) * p.heads * p.d * sizeof(T);
  const uint64_t out_head = p.d * sizeof(T);
  const bool turns = item < p.turned;  // else values that stay as they are
  const uint32_t first = item * V;
  float c[V], s[V];
  if (turns) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint32_t i = first + j;
      uint32_t axis = 0;
#pragma unroll
      for (int a = 0; a < G16_ROTARY_MAX_AXES - 1; ++a) axis += i >= p.ends[a];
      const double position = p.positions[static_cast<uint64_t>(axis) * p.rows + row];
      turn(position, p.freqs[i], c[j], s[j]);
    }
  }
  // Halves: V values from each of them; neighbours: 2 V values in a row. Those that stay are W in a row, as one such run or as two
  // (or as the same one twice).
  constexpr int L = NEIGHBOURS ? 1 : 2, N = 2 * V / L;
  const uint32_t stay = 2 * p.pairs + (item - p.turned) * W;
  const uint32_t at[2] = {static_cast<uint32_t>((turns ? (NEIGHBOURS ? 2 * first : first) : stay) * sizeof(T)),
                          static_cast<uint32_t>((turns ? p.pairs + first : stay + W - N) * sizeof(T))};
  for (uint32_t h0 = slice; h0 < p.heads; h0 += kAhead * p.slices) {
    Run<T, N> v[kAhead][L];
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      const uint32_t h = min(h0 + n * p.slices, p.heads - 1);
#pragma unroll
      for (int i = 0; i < L; ++i) v[n][i] = *reinterpret_cast<const Run<T, N>*>(x + h * p.x_head + at[i]);
    }
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      const uint32_t h = h0 + n * p.slices;
      if (h >= p.heads) break;
      if (turns) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          T& a = NEIGHBOURS ? v[n][0].v[2 * j] : v[n][0].v[j];
          T& b = NEIGHBOURS ? v[n][0].v[2 * j + 1] : v[n][L - 1].v[j];
          const float x0 = to_f(a), x1 = to_f(b);
          a = static_cast<T>(fmaf(x0, c[j], -(x1 * s[j])));
          b = static_cast<T>(fmaf(x1, c[j], x0 * s[j]));
        }
      }
#pragma unroll
      for (int i = 0; i < L; ++i) *reinterpret_cast<Run<T, N>*>(out + h * out_head + at[i]) = v[n][i];
    }
  }
}

template <typename T, int V, bool NEIGHBOURS>
int run(Params p, hipStream_t stream) {
  constexpr uint32_t W = 2 * V < 8 ? 2 * V : 8;
  p.turned = p.pairs / V;
  p.items = p.turned + (p.d - 2 * p.pairs) / W;
  // A thread for every head as long as that is few threads (a batch of tokens), then up to eight heads a thread.
  const uint64_t pieces = static_cast<uint64_t>(p.rows) * p.items;
  uint32_t each = 1;
  while (each < 8 && pieces * ((p.heads + each - 1) / each) > (1 << 19)) each *= 2;
  p.slices = (p.heads + each - 1) / each;
  const uint64_t blocks = (pieces * p.slices + kThreads - 1) / kThreads;
  if (blocks > (1u << 24) - 1) return G16_E_SHAPE;  // (2^32 threads a launch)
  return launch(rotary_kernel<T, V, NEIGHBOURS>, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), stream, p);
}
// Pairs of a thread: 16 bytes a load where their number allows that (neighbours: 12291 patches, 32 heads of 128 fp16, 40 pairs:
// 66 us with 32 bytes a thread, 60 so, and 40.8 with the values that stay in the same loop).
template <typename T>
int run(const Params& p, bool neighbours, hipStream_t stream) {
  constexpr uint32_t kMost = 16 / sizeof(T);
  if (!neighbours) {
    if (p.pairs % kMost == 0) return run<T, kMost, false>(p, stream);
    if (sizeof(T) == 2 && p.pairs % 4 == 0) return run<T, 4, false>(p, stream);
    return p.pairs % 2 == 0 ? run<T, 2, false>(p, stream) : run<T, 1, false>(p, stream);
  }
  if (p.pairs % (kMost / 2) == 0) return run<T, kMost / 2, true>(p, stream);
  if (sizeof(T) == 2 && p.pairs % 2 == 0) return run<T, 2, true>(p, stream);
  return run<T, 1, true>(p, stream);
}

// (what the Python binding packs)
static_assert(sizeof(g16_rotary_args) == 4 * 8 + 3 * 8 + 12 * 4, "no padding");

}  // namespace
}  // namespace g16

using namespace g16;

extern "C" int g16_rotary(const g16_rotary_args* args, void* stream) {
  if (args == nullptr) return G16_E_NULL;
  const g16_rotary_args& a = *args;
  if (a.is_f32 != 0 && a.is_f32 != 1) return G16_E_DTYPE;
  if (a.seqs < 0 || a.tokens < 0 || a.heads < 0 || a.d <= 0 || a.d % 8 != 0 || a.d > G16_ROTARY_MAX_D || a.pairs < 0 || 2 * a.pairs > a.d ||
      a.axes < 1 || a.axes > G16_ROTARY_MAX_AXES || (a.interleaved != 0 && a.interleaved != 1))
    return G16_E_SHAPE;
  int64_t pairs = 0;
  for (int i = 0; i < a.axes; ++i) {
    if (a.sections[i] < 0) return G16_E_SHAPE;
    pairs += a.sections[i];
  }
  if (pairs != a.pairs) return G16_E_SHAPE;
  if (a.seqs == 0 || a.tokens == 0 || a.heads == 0) return G16_OK;
  const int64_t rows = static_cast<int64_t>(a.seqs) * a.tokens, size = a.is_f32 ? 4 : 2;
  if (rows > (1LL << 31) - 1) return G16_E_SHAPE;
  if (a.x == nullptr || a.out == nullptr || (a.pairs > 0 && (a.positions == nullptr || a.freqs == nullptr))) return G16_E_NULL;
  if (!aligned16(a.x) || !aligned16(a.out) || a.x_seq * size % 16 != 0 || a.x_token * size % 16 != 0 || a.x_head * size % 16 != 0) return G16_E_ALIGN;
  Params p = {};
  p.x = static_cast<const char*>(a.x);
  p.out = static_cast<char*>(a.out);
  p.positions = a.positions;
  p.freqs = a.freqs;
  p.x_seq = a.x_seq * size;
  p.x_token = a.x_token * size;
  p.x_head = a.x_head * size;
  p.rows = static_cast<uint32_t>(rows);
  p.tokens = static_cast<uint32_t>(a.tokens);
  p.heads = static_cast<uint32_t>(a.heads);
  p.d = static_cast<uint32_t>(a.d);
  p.pairs = static_cast<uint32_t>(a.pairs);
  uint32_t end = 0;
  for (int i = 0; i < G16_ROTARY_MAX_AXES - 1; ++i) {
    end = i < a.axes ? end + static_cast<uint32_t>(a.sections[i]) : p.pairs;
    p.ends[i] = end;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  return a.is_f32 ? run<float>(p, a.interleaved != 0, s) : run<_Float16>(p, a.interleaved != 0, s);
}
