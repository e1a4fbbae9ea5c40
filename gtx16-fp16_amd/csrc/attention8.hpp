// The own keys of single tokens in a cache of 8 bits: what attention.hip calls of attention8.hip.
#pragma once

#include "attention_parts.hpp"

namespace g16 {

constexpr int kXcds = 8;
constexpr int kTile8 = 64;  // keys of a tile
constexpr int kWhole8 = 8;  // tiles of a request whose keys are never split

// n / by without a division: (2 n magic >> 32) >> shift, for n below 2^31.
struct Divide {
  uint32_t by, magic, shift;
  __device__ uint32_t operator()(uint32_t n) const { return __umulhi(2 * n, magic) >> shift; }
};
inline Divide divide_by(uint32_t by) {
  uint32_t shift = 0;
  while ((1ull << shift) < by) ++shift;
  return Divide{by, static_cast<uint32_t>((1ull << (31 + shift)) / by + 1), shift};
}

struct Params8 {
  const float *ks, *vs;
  int64_t ks_seq, ks_head, ks_tok, vs_seq, vs_head, vs_tok;  // elements
  int64_t k_tok, v_tok;                                      // bytes
  Divide page;
  int shares;    // at most
  bool split;    // shares of equal length; else one for each request
  int srt;       // rows of the shared keys' slots
  size_t first;  // floats of the shared keys' slots, before the own keys'
};

// Query rows that a workgroup has room for.
constexpr int rows_of8(int group) { return group == 1 ? 1 : group <= 4 ? 4 : group <= 8 ? 8 : group <= 16 ? 16 : 32; }
// Workgroups on a CU that the registers are held to.
constexpr int waves_of8(bool f32, int dp, int rows, bool full) {
  if (rows == 32) return dp == 64 ? 2 : 1;
  return f32 || dp == 128 || rows == 16 ? 2 : rows == 1 && full ? 4 : 3;
}

// Enqueues the products of the requests' own keys and the joins.
int run_own8(const Params& p, const Params8& e, int code, bool f32, hipStream_t stream);

}  // namespace g16
