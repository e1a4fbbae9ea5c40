// What the attention kernels of attention.hip and attention8.hip share: types and products, scores, the slots of partial sums,
// and the parts that the keys of single tokens are dealt in.
#pragma once

#include <cfloat>
#include <type_traits>

#include "code8.hpp"

namespace g16 {

typedef float float8v __attribute__((ext_vector_type(8)));

constexpr float kLag = 7.f;
// Where the largest score is more than this, the scores are rounded, like the maximum, before it is taken off them: the product with
// the scale within the difference, which is exact, would leave the best key's weight at 2 to the maximum's rounding.
constexpr float kWide = 0x1p22f;
// fp16 weights are 2^kShift above their value, by way of the exponent. fp32 ones would lose bits of the exponent by that
// (2^-20 of a weight at 23), and are multiplied by kScale: at most 2^-16, so that the sums over 65536
// keys of the largest weight stay within the values' range.
template <typename T>
constexpr float kShift = sizeof(T) == 2 ? 8.f : 0.f;
template <typename T>
constexpr float kScale = sizeof(T) == 2 ? 1.f : 0x1p-23f;
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kPlainCap = 256.f;  // largest tanh cap that fp16 inputs take the plain form for (tanh_of)
constexpr float kNoCap = 0x1p100f;  // a cap from here on changes no fp32 score below 2^88, and would not fit in log2 units
constexpr int kRowTile = 128, kKeyTile = 32;  // query rows of the two workgroup shapes
constexpr int kThreads = 256;

__device__ __attribute__((aligned(16))) const uint32_t g_zero_row[G16_ATTENTION_MAX_D] = {};

template <typename T>
struct Vec8 {
  using V = half8;
};
template <>
struct Vec8<float> {
  using V = float8v;
};

__device__ inline float16v mma(half8 a, half8 b, float16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ inline float16v mma(float8v a, float8v b, float16v c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// fp32 as three bf16 parts, hi + mid + lo.
typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bhalf2 __attribute__((ext_vector_type(2)));
struct Split8 {
  bhalf8 hi, mid, lo;
};
__device__ inline float16v mma(bhalf8 a, bhalf8 b, float16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ inline float8v widen(bhalf8 v) { return __builtin_convertvector(v, float8v); }
__device__ inline float8v whole(const Split8& s) { return widen(s.hi) + widen(s.mid) + widen(s.lo); }  // (no part rounds)
// ... all products of parts but the largest
__device__ inline float16v mma_small(const Split8& a, const Split8& b, float16v c) {
  c = mma(a.lo, b.hi, c);
  c = mma(a.mid, b.mid, c);
  c = mma(a.hi, b.lo, c);
  c = mma(a.mid, b.hi, c);
  return mma(a.hi, b.mid, c);
}
__device__ inline float16v mma(const Split8& a, const Split8& b, float16v c) { return mma(a.hi, b.hi, mma_small(a, b, c)); }
// What becomes of 8 values that are multiplied: fp16 as it is, fp32 in parts.
__device__ inline half8 operand(half8 v) { return v; }
// Values rounded to bf16, taken off them: 20 instructions for 8. (A dot product with (-1, 0) would save the unpacking,
// but v_dot2_f32_bf16 does not give the difference exactly, and takes as long.)
__device__ inline bhalf8 take_part(float8v& v) {
  bhalf8 part;
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const bhalf2 two = __builtin_convertvector((float2v{v[j], v[j + 1]}), bhalf2);
    const uint32_t bits = __builtin_bit_cast(uint32_t, two);
    part[j] = two[0];
    part[j + 1] = two[1];
    v[j] -= __uint_as_float(bits << 16);
    v[j + 1] -= __uint_as_float(bits & 0xffff0000u);
  }
  return part;
}
__device__ inline Split8 operand(float8v v) {
  Split8 s;
  s.hi = take_part(v);
  s.mid = take_part(v);
  s.lo = __builtin_convertvector(v, bhalf8);
  return s;
}
// The same for any fp32 value: whole() gives it back, NaN, infinities and those that round to one included.
__device__ inline Split8 operand_of_any(float8v v) {
  bhalf8 hi = __builtin_convertvector(v, bhalf8);
  float8v rest;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (fabsf(static_cast<float>(hi[j])) <= FLT_MAX || v[j] != v[j]) {
      rest[j] = v[j] - static_cast<float>(hi[j]);
    } else {  // its first 8 bits, cut off
      const float cut = __uint_as_float(__float_as_uint(v[j]) & 0xffff0000u);
      hi[j] = static_cast<__bf16>(cut);
      rest[j] = fabsf(cut) <= FLT_MAX ? v[j] - cut : 0.f;
    }
  }
  Split8 s = operand(rest);
  // (at most 16 bits are left: two parts)
  return Split8{hi, s.hi, s.mid};
}

template <typename P>
__device__ inline P* uniform(P* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
  return reinterpret_cast<P*>((static_cast<uint64_t>(hi) << 32) | lo);
}
__device__ inline int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Where part `i` of `parts` about equal ones of n things begins (32 bits throughout: n * i / parts in 64 would be
// 150 scalar instructions).
__device__ inline int share_begin(int n, int i, int parts) {
  const uint32_t each = static_cast<uint32_t>(n) / static_cast<uint32_t>(parts), more = static_cast<uint32_t>(n) % static_cast<uint32_t>(parts);
  return static_cast<int>(each * i + min(more, static_cast<uint32_t>(i)));
}

struct Params {
  const char *q, *k, *v, *sk, *sv;
  char* out;
  const int32_t *q_off, *k_off, *visible, *lengths, *pages;
  const float* slopes;
  float* part;
  int64_t q_seq, q_tok, q_head, k_seq, k_head, v_seq, v_head, sk_head, sv_head;  // bytes
  uint32_t k_tok, v_tok, sk_tok, sv_tok;                                        // bytes
  int seqs, q_len, k_len, hq, hkv, group, d, shared, causal;
  int page, max_pages, num_pages;
  int tiles, splits;              // prompts: row tiles (an upper bound where packed), key splits
  int stiles, ssplits;            // single tokens: row tiles and splits of the shared keys
  int otiles, oitems, least;      // ... row tiles of a request's `group` rows; parts of the own keys, of all
                                  // requests together: about `oitems`, of at least `least` tiles (0: one each)
  float scale, softcap;  // scale > 0, with its sign (0 for 0) in `sign`, which the queries take on
  float sign;
};

// Scores (products q.k) -> t = log2(e) * f(scale * s) - slope * distance, for keys pos0 + {0 .. } of a
// block whose lane half h holds keys 8 (r / 4) + 4 h + r % 4 in register r.
struct Scoring {
  float c;         // scale * log2(e)
  float cap;       // softcap * log2(e)
  float inv, inv2; // scale / softcap, and that times 2 log2(e)
  bool capped, fine, biased;  // fine: the cap needs tanh's relative precision near 0 (below)
};

__device__ inline Scoring scoring(const Params& p) {
  Scoring s;
  s.c = p.scale * kLog2e;
  s.capped = p.softcap != 0.f && p.softcap < kNoCap;
  s.fine = p.softcap > kPlainCap;
  s.biased = p.slopes != nullptr;
  s.cap = p.softcap * kLog2e;
  // (held to where no score's product with it is 0 times infinity; past that every score is at a cap of nearly 0)
  s.inv = s.capped ? fminf(p.scale / p.softcap, 1e37f) : 0.f;
  s.inv2 = s.inv * (2.f * kLog2e);
  return s;
}

// tanh to fp32's last bits near 0, where a cap leaves most scores (an odd polynomial fitted by least
// squares to (tanh(y) / y - 1) / y^2 on [0, 0.625], largest relative error 4e-9), and 1 - 2 / (e^2y + 1)
// past it. With fp16 inputs and a cap up to kPlainCap the second form's absolute error, 1e-7 of the cap, is
// enough throughout.
__device__ inline float tanh_of(float y) {
  const float e = __builtin_amdgcn_exp2f(y * (2.f * kLog2e));
  const float big = 1.f - 2.f * __builtin_amdgcn_rcpf(e + 1.f);
  const float u = y * y;
  float r = fmaf(u, -0.00571705f, 0.02065059f);
  r = fmaf(u, r, -0.0537435f);
  r = fmaf(u, r, 0.13331491f);
  r = fmaf(u, r, -0.33333284f);
  r = fmaf(y * u, r, y);
  return fabsf(y) < 0.625f ? r : big;
}

// ---- partial sums ----------------------------------------------------------------------------------------
// Where a tile's rows go: the output, or a slot of the workspace with rows x DP sums, then the rows'
// reference maxima and sums of weights (and a gap, so that every slot starts on 16 bytes).
__host__ __device__ constexpr size_t slot_floats(int rows, int dp) { return static_cast<size_t>(rows) * (dp + 4); }
struct Slot {
  float* at;  // NULL: the output
  int rows;
};
template <int DP>
__device__ inline float* slot_m(const Slot& s) { return s.at + static_cast<size_t>(s.rows) * DP; }

template <typename T, int N>
__device__ inline void store_out(char* out, int d0, const float (&v)[N]) {
  if constexpr (sizeof(T) == 2) {
    if constexpr (N == 4) {
      const half4 h = {static_cast<_Float16>(v[0]), static_cast<_Float16>(v[1]), static_cast<_Float16>(v[2]), static_cast<_Float16>(v[3])};
      *reinterpret_cast<half4*>(out + d0 * 2) = h;
    } else {
      half8 h;
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = static_cast<_Float16>(v[i]);
      *reinterpret_cast<half8*>(out + d0 * 2) = h;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<float4v*>(out + (d0 + i) * 4) = float4v{v[i], v[i + 1], v[i + 2], v[i + 3]};
  }
}

// 1 / l, with 0 for a row that saw no key (a NaN stays one)
__device__ inline float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }

// One row from its partial sums: `of(i)` gives part i's sums, reference maximum and, `rows` floats behind it,
// sum of weights. A wavefront a row: a lane holds 4 values of every kP-th part, whose weight the lane of
// that number has. The sums' loads do not wait for the weights.
// (join_sums: the same without the division, o being values 4 (lane % (DP / 4)) ..)
template <int DP, typename F>
__device__ inline void join_sums(int parts, const F& of, float& top, float& l, float4v& o) {
  constexpr int L = DP / 4, kP = kWave / L, kB = 8;  // lanes of a part, parts at a time, loads at a time
  const int lane = threadIdx.x & 63, d0 = (lane % L) * 4, mine = lane / L;
  const float *s, *m;
  int rows;
  float first_m = -__builtin_huge_valf(), first_l = 0.f;
  if (lane < parts) {
    of(lane, s, m, rows);
    first_m = *m;
    first_l = m[rows];
  }
  float4v v[kB];
  auto load = [&](int b) {
#pragma unroll
    for (int i = 0; i < kB; ++i) {
      of(min(b + i * kP + mine, parts - 1), s, m, rows);
      v[i] = *reinterpret_cast<const float4v*>(s + d0);
    }
  };
  load(0);
  top = first_m;
  for (int i = lane + kWave; i < parts; i += kWave) {
    of(i, s, m, rows);
    top = fmaxf(top, *m);
  }
#pragma unroll
  for (int i = 1; i < kWave; i *= 2) top = fmaxf(top, __shfl_xor(top, i));
  float f = 0.f;  // the weight of part (64 n + lane)
  l = 0.f;
  o = float4v{};
  for (int b = 0; b < parts; b += kB * kP) {
    if (b % kWave == 0) {
      float pm = first_m, pl = first_l;
      if (b > 0 && b + lane < parts) {
        of(b + lane, s, m, rows);
        pm = *m;
        pl = m[rows];
      }
      f = b + lane >= parts ? 0.f : (pm == top ? 1.f : __builtin_amdgcn_exp2f(pm - top));
      l = fmaf(f, b + lane < parts ? pl : 0.f, l);
    }
    if (b > 0) load(b);
#pragma unroll
    for (int i = 0; i < kB; ++i) {
      const int part = b + i * kP + mine;
      const float fi = __shfl(f, part & (kWave - 1));
      if (part < parts) o += fi * v[i];
    }
  }
#pragma unroll
  for (int i = 1; i < kWave; i *= 2) l += __shfl_xor(l, i);
#pragma unroll
  for (int i = L; i < kWave; i *= 2)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], i);
}
template <typename T, int DP, typename F>
__device__ inline void join_row(char* out, int d, int parts, const F& of) {
  const int lane = threadIdx.x & 63, d0 = lane % (DP / 4) * 4;
  float top, l;
  float4v o;
  join_sums<DP>(parts, of, top, l, o);
  const float inv = inverse(l);
  const float r[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
  if (lane < DP / 4 && d0 < d) store_out<T, 4>(out, d0, r);
}

// ---- the parts of single tokens' keys ----------------------------------------------------------------------
__host__ __device__ inline int own_rows(int group) { return group < kKeyTile ? group : kKeyTile; }

struct Part {
  int seq, len, split, splits;  // the request and its length; which of its parts this is, and of how many
  int first;                    // number of the request's first part
};
__device__ inline int length_of(const Params& p, int b) { return min(max(p.lengths[b], 0), p.k_len); }

// Tiles of 32 keys a part gets: the requests' tiles over the parts that there should be.
__device__ inline int part_tiles(const Params& p) {
  const int lane = threadIdx.x & 63;
  int64_t total = 0;
  for (int b = lane; b < p.seqs; b += kWave) total += ceil_div(length_of(p, b), 32);
#pragma unroll
  for (int i = 1; i < kWave; i *= 2) total += __shfl_xor(static_cast<long long>(total), i);
  return max(p.least, uniform(static_cast<int>((total + p.oitems - 1) / p.oitems)));
}
// Part `item` of all (by_item), or the first part of request `item`. false: past the last one.
__device__ inline bool find_part(const Params& p, int item, bool by_item, Part& r) {
  if (p.least == 0) {
    r = Part{item, item < p.seqs ? uniform(length_of(p, item)) : 0, 0, 1, item};
    return item < p.seqs;
  }
  const int lane = threadIdx.x & 63, chunk = part_tiles(p);
  int before = 0;
  for (int b0 = 0; b0 < p.seqs; b0 += kWave) {
    const int b = b0 + lane, len = b < p.seqs ? length_of(p, b) : 0;
    const int n = b < p.seqs ? max(1, ceil_div(ceil_div(len, 32), chunk)) : 0;
    int upto = n;
#pragma unroll
    for (int i = 1; i < kWave; i *= 2) {
      const int x = __shfl_up(upto, i);
      if (lane >= i) upto += x;
    }
    const uint64_t hit = __ballot(by_item ? item < before + upto : b == item);
    if (hit != 0) {
      const int l = __builtin_ctzll(hit);
      r.seq = b0 + l;
      r.len = __builtin_amdgcn_readlane(len, l);
      r.splits = __builtin_amdgcn_readlane(n, l);
      r.first = before + __builtin_amdgcn_readlane(upto, l) - r.splits;
      r.split = by_item ? item - r.first : 0;
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, kWave - 1);
  }
  return false;
}

}  // namespace g16
