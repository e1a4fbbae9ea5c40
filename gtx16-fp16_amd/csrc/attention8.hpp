// The own keys of single tokens in a cache of 8 bits: what attention.hip calls of attention8.hip.
#pragma once

#include "attention_parts.hpp"

namespace g16 {

constexpr int kXcds = 8;

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
  int parts;     // of all requests, at most
  size_t first;  // floats of the shared keys' slots, before these parts'
};

// Enqueues the products of the requests' own keys.
int run_own8(const Params& p, const Params8& e, int code, bool f32, hipStream_t stream);

}  // namespace g16
