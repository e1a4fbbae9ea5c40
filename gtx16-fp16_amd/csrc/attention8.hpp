// The own keys of single tokens in a cache of 8 bits: what attention.hip calls of attention8.hip.
#pragma once

#include "attention_parts.hpp"

namespace g16 {

constexpr int kXcds = 8;
constexpr int kTile8 = 64;  // keys of a tile
constexpr int kWhole8 = 8;  // tiles of a request whose keys are never split
constexpr int kHeads8 = 4;  // key heads that a workgroup may take together,
// of how many query rows at most (16, 64 heads on 4 of 128: 40 requests of up to 8192 56.7 us, by single heads 61.4, but 64 of up to 700
// 25.4 and 22.8; 8, 64 heads on 8: 82.4 and 94.4, 25.8 and 31.2)
constexpr int kRowsOfHeads8 = 8;

// A request's slots: the first one's number, and how many there are.
struct Slots {
  int first, count;
};

struct Params8 {
  const float *ks, *vs;
  int64_t ks_seq, ks_head, ks_tok, vs_seq, vs_head, vs_tok;  // elements
  int64_t k_tok, v_tok;                                      // bytes
  Divide page;
  int heads;     // key heads of a workgroup, 1 or kHeads8
  int shares;    // at most
  bool split;    // shares of equal length; else one for each request
  int srt;       // rows of the shared keys' slots
  bool apart;    // the own keys have a launch of their own
  size_t first;  // floats of the shared keys' slots, before the own keys'
  Slots* table;  // of all requests, for the join (NULL: there is none), before the slots
};

// Query rows that a workgroup has room for.
constexpr int rows_of8(int group) { return group == 1 ? 1 : group <= 4 ? 4 : group <= 8 ? 8 : group <= 16 ? 16 : 32; }
// Workgroups on a CU that the registers are held to: as many as leave a tile's keys and values in registers. (One more for heads of
// 128, and some are in scratch memory: 106 us where two take 87, 40 requests of up to 8192 e4m3 keys by single heads. fp32's 8 and 16 rows of
// 128 and 32 of 64 have 12 to 144 bytes of a lane there, and are slower by one workgroup all the same: 58.8 us for 53.4, 32 heads on
// 2 of 128, and 63.7 for 58.2, 40 on 2 of 64, 40 requests of up to 8192.) Three for fp16 heads of 64: two take 49.6 us where
// three take 45.7, 96 requests of up to 2048, 12 heads ordered by heads, but with four heads together 45.8 for 46.6, and 49.7 for
// 51.2, 40 of up to 8192, 32 heads on 8; four 48.3 and 51.4.
constexpr int waves_of8(bool f32, int dp, int rows) {
  if (rows == 32) return dp == 64 ? 2 : 1;
  return f32 || dp == 128 || rows == 16 ? 2 : 3;
}

inline unsigned workgroups_of8(const Params& p, const Params8& e) {
  return static_cast<unsigned>(e.shares >= kXcds ? ceil_div(e.shares, kXcds) * kXcds : e.shares) * p.otiles * (p.hkv / e.heads);
}

// Enqueues the products of the requests' own keys, where they are apart, and the joins.
int run_own8(const Params& p, const Params8& e, int code, bool f32, hipStream_t stream);

}  // namespace g16
