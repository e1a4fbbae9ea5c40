// Single tokens over a cache of 8 bits (g16_attention_decode8; its formulas stand in g16.h): the products of the requests' own
// keys, by one workgroup. A shared prefix is not in 8 bits and shared_workgroup's (attention.hip), the joins are attention8.hip's.
//
// All requests' keys, in tiles of 64 one request after another, are dealt in shares of equal length, as many as run on the card at
// once: whatever the lengths, all workgroups end together (see Deal for few keys). A workgroup has the query rows of one key head and a
// share's tiles, a request's after another's; its four wavefronts take a tile in turn (or a head each, see own8_workgroup),
// straight from memory into registers:
//   * S = Q K^T in 16x16x32 blocks of 16 keys, lane l's key l % 16, by way of LDS. A step's values of a lane are half of a 16-byte
//     piece, in another order than in memory, the queries' too.
//   * With few query rows the blocks' 16 rows are as many copies of them, and the lanes of row group l / 16 keep those of
//     another block of keys: up to four rows, lane l has the scores of key l of the tile, and a row's 64 weights are one
//     register; up to eight, two blocks share a register set. What a score costs (an exponential, the parts of its
//     weight) is paid for RQ rows, not 16.
//   * O^T += V^T P^T, 32 keys a step: the weights go through LDS, from where lane l takes those of query row l % 16 and keys
//     8 (l / 16) + {0..7}. It loads DP / 16 values of each of these eight keys, from value (l % 16) DP / 16 on: a key's values are
//     one run of an instruction. Byte b of the eight loads makes the operand of block b, so the transposition costs
//     nothing but the choice of bytes, and block b's row m is value m DP / 16 + b.
//   * Codes are exact in fp16 and bf16. K is multiplied as fp16 where the queries are, else as bf16 with the queries in three
//     parts. A key's scale joins its score; a value's joins its weight, whose range then is fp32's, so weights are multiplied as
//     bf16 parts: two for fp16 (to 2^-17; results are 2.1e-4 from the exact ones, all of it their own rounding, and 2.6e-4 after a
//     shared prefix, whose weights shared_workgroup rounds to fp16, as for 16 bits), three for fp32.
//     So that the last of three is no subnormal, which the products take for 0, a row's fp32 sums are kept in a unit of its own, a
//     power of two that brings its largest product of weight and scale to 2^60 or so, and all down to 2^-170 of it have
//     their bits: it falls where a product is past 2^80, and rises as far as a new maximum makes the sums fall. (With one unit
//     for all rows, by the largest scale, rows that gave a value 2^60 times the others' no weight lost their result.)
//   * The keys' registers are loaded again as soon as the first product has read them, the values' after the second;
//     other wavefronts fill the gaps. The places of a tile's rows are found one key a lane and passed on through LDS.
// A key behind its part's end, or on a page outside the cache, is read from a row of zeros; the former get no weight.
#pragma once

#include "attention8.hpp"

namespace g16 {
namespace {

__device__ inline float4v mma16(half8 a, half8 b, float4v c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ inline float4v mma16(bhalf8 a, bhalf8 b, float4v c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

__device__ inline uint32_t high_halves(float a, float b) {  // bf16 of two numbers that it holds exactly
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

// Eight codes in a row as fp16, exactly.
template <int CODE>
__device__ inline half8 halves(u32x2 codes) {
  u32x4 r;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    if constexpr (CODE == G16_CODE_INT8) {
      // 0x6400 | (code + 128) is 1024 + 128 + code
      const uint32_t u = codes[w] ^ 0x80808080u;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t two = __builtin_amdgcn_perm(0x64646464u, u, j == 0 ? 0x07010700u : 0x07030702u);
        r[2 * w + j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, two) - half2v{1152.f16, 1152.f16});
      }
    } else {
      r[2 * w] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[w], 1.f, false));
      r[2 * w + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[w], 1.f, true));
    }
  }
  return __builtin_bit_cast(half8, r);
}
// ... as bf16
template <int CODE>
__device__ inline bhalf8 bfloats(u32x2 codes) {
  float x[8];
  decode8<CODE>(codes, x);
  return __builtin_bit_cast(bhalf8, (u32x4{high_halves(x[0], x[1]), high_halves(x[2], x[3]), high_halves(x[4], x[5]), high_halves(x[6], x[7])}));
}
// Byte `b` of eight dwords as bf16.
template <int CODE>
__device__ inline bhalf8 bfloats_of_byte(const uint32_t (&v)[8], int b) {
  u32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (CODE == G16_CODE_INT8) {
      r[j] = high_halves(static_cast<float>(static_cast<int8_t>(v[2 * j] >> (8 * b))), static_cast<float>(static_cast<int8_t>(v[2 * j + 1] >> (8 * b))));
    } else {
      const uint32_t two = __builtin_amdgcn_perm(v[2 * j + 1], v[2 * j], 0x0c0c0400u + 0x0101u * b);
      r[j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(two, 1.f, false));
    }
  }
  return __builtin_bit_cast(bhalf8, r);
}

template <typename T>
struct Query8;
template <>
struct Query8<_Float16> {
  half8 v;
  __device__ void set(half8 x) { v = x; }
  template <int CODE>
  __device__ float4v times(u32x2 codes, float4v c) const {
    return mma16(v, halves<CODE>(codes), c);
  }
};
template <>
struct Query8<float> {
  Split8 v;
  __device__ void set(float8v x) { v = operand_of_any(x); }
  // (the small products first: each one added to the large ones' sum would round it)
  template <int CODE>
  __device__ float4v times(u32x2 codes, float4v c) const {
    const bhalf8 k = bfloats<CODE>(codes);
    return mma16(v.hi, k, mma16(v.mid, k, mma16(v.lo, k, c)));
  }
};

template <typename V>
__device__ inline V load_at(uint64_t address) {  // (by a pointer of no address space the loads would count as LDS's, too)
  return *reinterpret_cast<const __attribute__((address_space(1))) V*>(address);
}

// LDS of one lane group is written and read by the same wavefront, in its order.
__device__ inline void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

constexpr int kRun8 = kTile8 + 8;  // weights of a row in LDS: rows on different banks

// ---- shares ----------------------------------------------------------------------------------------------
// A request without keys has one tile, too: somebody has to write its zeros. (The host sees to it that 32 bits hold all tiles.)
__device__ inline int tiles_of(int len) { return max(1, ceil_div(len, kTile8)); }

// The sum of a value over the lanes up to and with this one.
__device__ inline int sum_up(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // within rows of 16 lanes: from 1, 2, 4 and 8 before
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // rows 1 and 3: the last lane's of the row before
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // rows 2 and 3: lane 31's
  return v;
}

// A run of 64 requests in a wavefront: lane i has the length of request b0 + i and how many of what is counted (tiles, or pieces
// of `chunk` tiles) there are up to and with its own.
struct Run64 {
  int len, count, upto;
  __device__ Run64(const Params& p, int b0, int chunk = 1) {
    const int lane = threadIdx.x & 63;
    len = b0 + lane < p.seqs ? length_of(p, b0 + lane) : 0;
    set(b0 + lane < p.seqs, chunk);
  }
  __device__ void set(bool some, int chunk) {
    count = some ? tiles_of(len) : 0;
    if (chunk > 1) count = static_cast<int>(static_cast<uint32_t>(count + chunk - 1) / static_cast<uint32_t>(chunk));
    upto = sum_up(count);
  }
  __device__ int all() const { return __builtin_amdgcn_readlane(upto, kWave - 1); }
};
__device__ inline int all_tiles(const Params& p, const Run64& head) {
  int total = head.all();
  for (int b0 = kWave; b0 < p.seqs; b0 += kWave) total += Run64(p, b0).all();
  return total;
}

// How all requests' tiles are dealt. Long ones in shares of equal length, whatever the requests: the first `more` shares
// have each + 1, the others each. Where a share would have few tiles, its time is that of the waits for one after another, not of its bytes,
// and a second request's would come on top: every request then has its own pieces, of `chunk` tiles, one for each
// wavefront or two (16 requests of up to 1500, 32 heads on 8 of 128, HEADS = 1: 24.0 us by shares, 20.9 so; HEADS = 4: 20.1 and 20.9,
// but 64 of up to 700 25.3 and 24.5).
struct Deal {
  int shares = 1, each = 1, more = 0, chunk = 0;
  __device__ Deal() {}
  __device__ Deal(const Params& p, const Params8& e, int total) {
    const uint32_t waves = 4 / e.heads;  // wavefronts that a head has
    const int each_one = static_cast<int>((static_cast<uint32_t>(total) + 2u * p.seqs) / (waves * e.shares)) + 1;
    chunk = each_one <= 2 ? static_cast<int>(waves) * each_one : 0;
    shares = e.shares;
    each = static_cast<int>(static_cast<uint32_t>(total) / static_cast<uint32_t>(shares));
    more = total - each * shares;
  }
  __device__ int begin(int share) const { return each * share + min(more, share); }
  __device__ int share_of(int tile) const {
    const int ahead = more * (each + 1);
    return tile < ahead ? static_cast<int>(static_cast<uint32_t>(tile) / static_cast<uint32_t>(each + 1))
                        : more + static_cast<int>(static_cast<uint32_t>(tile - ahead) / static_cast<uint32_t>(each));
  }
};

// What a workgroup has: `tiles` tiles from one of request `seq` on, over the requests behind it as well; then, of pieces, the one
// `shares` further on.
struct Share {
  int seq, len, tile, tiles, slot;  // the first request, its length, the first tile of it; the first slot
  int ahead;                        // tiles of the requests before that one
  bool pieces;
};
// Piece number `piece` (a share is one).
__device__ inline bool find_share(const Params& p, const Params8& e, int piece, Share& r, Deal& deal) {
  r.pieces = false;
  r.ahead = 0;
  if (!e.split) {
    if (piece >= p.seqs) return false;
    r.seq = r.slot = piece;
    r.len = uniform(length_of(p, piece));
    r.tile = 0;
    r.tiles = tiles_of(r.len);
    return true;
  }
  Run64 head(p, 0);
  deal = Deal(p, e, all_tiles(p, head));
  r.pieces = deal.chunk > 0;
  const int from = r.pieces ? piece : deal.begin(piece);
  if (!r.pieces) r.tiles = deal.begin(piece + 1) - from;
  if (r.pieces ? false : piece >= deal.shares || r.tiles == 0) return false;
  if (r.pieces) head.set(static_cast<int>(threadIdx.x & 63) < p.seqs, deal.chunk);
  int before = 0;
  for (int b0 = 0; b0 < p.seqs; b0 += kWave) {
    const Run64 run = b0 == 0 ? head : Run64(p, b0, r.pieces ? deal.chunk : 1);
    const uint64_t hit = __ballot(from < before + run.upto);
    if (hit != 0) {
      const int at = __builtin_ctzll(hit), behind = from - before - __builtin_amdgcn_readlane(run.upto - run.count, at);
      r.seq = b0 + at;
      r.len = __builtin_amdgcn_readlane(run.len, at);
      r.tile = r.pieces ? behind * deal.chunk : behind;
      if (r.pieces) r.tiles = min(deal.chunk, tiles_of(r.len) - r.tile);
      r.slot = r.pieces ? piece : piece + r.seq;
      r.ahead = from - r.tile;
      return true;
    }
    before += run.all();
  }
  return false;
}
// RQ: query rows that there is room for, 1, 4, 8, 16 or 32. FULL: heads of DP values.
template <typename T, int DP, int RQ>
struct Shape8 {
  static constexpr int QP = RQ <= 4 ? 4 : RQ == 8 ? 8 : 16;  // rows of a block that are one copy
  static constexpr int NR = RQ == 32 ? 2 : 1;                // blocks of rows
  static constexpr int R = RQ;
  static constexpr int NS = QP / 4;             // register sets of scores a block of rows has
  static constexpr int RI = RQ < 4 ? RQ : 4;    // registers of a set in use
  static constexpr int PARTS = sizeof(T) == 4 ? 3 : 2;
};

// What a workgroup keeps in LDS: its wavefronts' keys and weights, which the sums that are joined take the place of; the places of
// a tile's rows, of keys and of values; maxima and sums.
template <typename T, int NR>
struct Lifts {};
template <int NR>
struct Lifts<float, NR> {
  float lifts[4][16 * NR];  // of a wavefront's rows: what large queries have been divided by
};
template <typename T, int DP, int RQ>
struct Lds8 : Lifts<T, Shape8<T, DP, RQ>::NR> {
  using S = Shape8<T, DP, RQ>;
  static constexpr int kKeys = kTile8 * DP, kWeights = S::PARTS * S::R * kRun8 * 2, kSums = S::R * DP * 4;  // bytes of a wavefront
  alignas(16) char data[4 * (kKeys + kWeights > kSums ? kKeys + kWeights : kSums)];
  alignas(16) uint64_t places[4][2][kTile8];
  float joint[2][4][S::R];
};

// Workgroup `block` of those for the requests' own keys. HEADS: 1, a key head, whose tiles the wavefronts take in turn; or 4, one for
// each wavefront, which has all of the share's tiles. What a workgroup reads of a token is then four heads' codes in
// a row, and their scales: 40 requests of up to 8192 e4m3 keys, 32 heads on 8 of 128, take 72.7 us, with HEADS = 1 85.8;
// 96 of up to 2048, 12 heads of 64, 46.6 and 54.7. No wavefront waits for another, there is nothing to join in LDS, and a
// row has four times as many parts. A cache that is ordered by heads has a head's codes in a row, and HEADS = 1.
template <typename T, int DP, int CODE, int RQ, bool FULL, int HEADS>
__device__ inline void own8_workgroup(const Params& p, const Params8& e, int block, Lds8<T, DP, RQ>& shared) {
  using S = Shape8<T, DP, RQ>;
  constexpr int VB = DP / 16, VW = DP / 64;  // values of a lane, and blocks of the second product; dwords of a lane's values
  constexpr int R = S::R, NR = S::NR, NS = S::NS, RI = S::RI, PARTS = S::PARTS;
  constexpr int kKeys = Lds8<T, DP, RQ>::kKeys, kWeights = Lds8<T, DP, RQ>::kWeights;
  char* lds = shared.data;
  auto& places = shared.places;
  auto& joint = shared.joint;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 15, g = lane >> 4;
  // Workgroups go to the XCDs in turn, and every XCD has an L2 of its own. The heads of a share read the same cache lines (of
  // codes where a head's are less than a line, of scales always), so they are all given to one XCD where there are shares for all
  // (96 requests of up to 2048, 12 heads of 64, by single heads: 76 us, and by this alone 63; four heads together take as long without).
  int lin = block;
  if (e.shares >= kXcds) {
    const int per = p.otiles * (p.hkv / HEADS), i = lin / kXcds, share = i / per * kXcds + lin % kXcds;
    if (share >= e.shares) return;
    lin = share * per + i % per;
  }
  const int kv = HEADS == 1 ? lin % p.hkv : lin % (p.hkv / HEADS) * HEADS + wave;
  lin /= p.hkv / HEADS;
  const int rt = lin % p.otiles, share = lin / p.otiles;
  Share has;
  Deal deal;
  if (!find_share(p, e, share, has, deal)) return;
  const int orows = own_rows(p.group);
  const Scoring sc = scoring(p);
  int b = has.seq, len = has.len, u0 = has.tile, todo = has.tiles;  // request, its first tile here, tiles to do
  int at_slot = has.slot, ahead = has.ahead;

  for (int piece = share;;) {
    const int tiles = tiles_of(len), u1 = min(u0 + todo, tiles);
    const int begin = kTile8 * u0, end = min(len, kTile8 * u1);

    // ---- places of a tile's rows, this lane's key ----
    const int32_t* table = p.pages == nullptr ? nullptr : p.pages + static_cast<size_t>(b) * p.max_pages;
    const char *kbase = p.k + kv * p.k_head, *vbase = p.v + kv * p.v_head;
    const float *ksbase = e.ks + kv * e.ks_head, *vsbase = e.vs + kv * e.vs_head;
    auto page_of = [&](int j0) {  // -1: no such key
      const int j = j0 + lane;
      int pg = -1;
      if (j < end) {
        pg = b;
        if (table != nullptr) {
          pg = table[e.page(j)];
          if (static_cast<unsigned>(pg) >= static_cast<unsigned>(p.num_pages)) pg = -1;
        }
      }
      return pg;
    };
    float ks, vs;  // of this lane's key
    auto find = [&](int j0, int pg) {
      const int j = j0 + lane, at = table != nullptr ? j - e.page(j) * e.page.by : j;
      const uint64_t zero = reinterpret_cast<uint64_t>(g_zero_row);
      places[wave][0][lane] = pg < 0 ? zero : reinterpret_cast<uint64_t>(kbase + pg * p.k_seq + at * e.k_tok);
      places[wave][1][lane] = pg < 0 ? zero : reinterpret_cast<uint64_t>(vbase + pg * p.v_seq + at * e.v_tok);
      ks = pg < 0 ? 0.f : ksbase[pg * e.ks_seq + at * e.ks_tok];
      vs = pg < 0 ? 0.f : vsbase[pg * e.vs_seq + at * e.vs_tok];
      wave_order();
    };
    // A key is CH pieces of 16 bytes. A load takes whole keys, in the order in which they lie in memory; LDS turns them
    // into the product's order, where lane l has piece 4 c + l / 16 of key l % 16: pieces are at places that put those of 8 keys on
    // different banks. (Loaded in that order, a lane's piece next to another key's, 40 requests of 8192 e4m3 keys of 8 heads of 128
    // take 166 us, so 161 (HEADS = 1); ordered by heads 143 and 146.)
    constexpr int CH = DP / 16, PER = 64 / CH, NK = CH;  // pieces of a key; keys of a load; loads of a tile
    auto place_of = [](int key, int piece) { return key * DP + ((piece ^ (CH == 8 ? key & 7 : (key >> 1) & 3)) << 4); };
    char* keys = lds + wave * (kKeys + kWeights);
    u32x4 k[NK];
    uint32_t v[2][8][VW];
    auto load_k = [&]() {
      typedef uint32_t piece __attribute__((ext_vector_type(4), aligned(8)));
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        const uint64_t row = places[wave][0][n * PER + lane / CH];
        const int at0 = lane % CH * 16;
        if constexpr (FULL) {
          k[n] = load_at<piece>(row + at0);
        } else {  // (rows end at a multiple of 8, and nothing behind them is read)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const bool some = at0 + 8 * h < p.d;
            const u32x2 x = load_at<u32x2>(row + (some ? at0 + 8 * h : 0));
            k[n][2 * h] = some ? x[0] : 0;
            k[n][2 * h + 1] = some ? x[1] : 0;
          }
        }
      }
    };
    auto load_v = [&]() {
      const bool some = FULL || col * VB < p.d;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint64_t row = places[wave][1][32 * s + 8 * g + i] + (some ? col * VB : 0);
          if constexpr (VW == 2) {
            const u32x2 x = load_at<u32x2>(row);
            v[s][i][0] = some ? x[0] : 0;
            v[s][i][1] = some ? x[1] : 0;
          } else {
            const uint32_t x = load_at<uint32_t>(row);
            v[s][i][0] = some ? x : 0;
          }
        }
    };

    if (u0 == 0 && kv == 0 && rt == 0 && e.table != nullptr && tid == 0) {
      Slots s = {at_slot, 1};
      if (has.pieces) s.count = static_cast<int>(static_cast<uint32_t>(tiles + deal.chunk - 1) / static_cast<uint32_t>(deal.chunk));
      else if (e.split) s.count = deal.share_of(ahead + tiles - 1) - share + 1;
      e.table[b] = s;
    }

    int j0 = begin + (HEADS == 1 ? kTile8 * wave : 0);
    constexpr int kStep = 4 / HEADS * kTile8;
    if (j0 < end) {
      find(j0, page_of(j0));
      load_k();
      load_v();
    }
    int next = page_of(j0 + kStep);

    // ---- query rows ----
    // This lane's rows of the scores, 16 r + mine + i; of a set s of them this lane's key is key_of(s).
    const int mine = S::QP == 4 ? 0 : S::QP == 8 ? 4 * (g & 1) : 4 * g;
    auto key_of = [&](int s) { return S::QP == 4 ? lane : S::QP == 8 ? 32 * s + 16 * (g >> 1) + col : 16 * s + col; };
    Query8<T> q[NR][DP / 32];
    constexpr bool kUnits = sizeof(T) == 4;
    constexpr float kMostUnit = 0x1p100f, kLarge = 0x1p64f;
    float slope[NR][RI], m[NR][RI], l[NR][RI], unit[NR][RI];
    float4v o[NR][VB];
    bool lifted = false;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int row = rt * kKeyTile + 16 * r + col % S::QP;
      const bool some = row < p.group;
      const char* at = p.q + b * p.q_seq + (kv * p.group + (some ? row : 0)) * p.q_head;
      bool large = false;
#pragma unroll
      for (int s = 0; s < DP / 32; ++s) {
        using V8 = typename Vec8<T>::V;
        const int d0 = 64 * (s >> 1) + 16 * g + 8 * (s & 1);
        V8 x = {};
        if (some && d0 < p.d) x = *reinterpret_cast<const V8*>(at + d0 * sizeof(T));
        if (p.sign != 1.f) x *= static_cast<T>(p.sign);
        if constexpr (kUnits) {
#pragma unroll
          for (int j = 0; j < 8; ++j) large = large || fabsf(x[j]) >= kLarge;
        }
        q[r][s].set(x);
      }
      if constexpr (kUnits) {
        // The sums of a large query's products with codes, which the keys' scales may well bring back, could be past fp32's
        // range: it is divided, and its scores multiplied once they have their scales.
        const uint64_t lanes = __ballot(large);
        if (lanes != 0) {
          const bool divided = ((lanes | lanes >> 16 | lanes >> 32 | lanes >> 48) >> col & 1) != 0;
#pragma unroll
          for (int s = 0; s < DP / 32; ++s) {
            const int d0 = 64 * (s >> 1) + 16 * g + 8 * (s & 1);
            float8v x = {};
            if (some && d0 < p.d) x = *reinterpret_cast<const float8v*>(at + d0 * 4);
            q[r][s].set(x * (divided ? p.sign / kLarge : p.sign));
          }
          if (NR > 1 && !lifted) shared.lifts[wave][16 * (1 - r) + col] = 1.f;
          shared.lifts[wave][16 * r + col] = divided ? kLarge : 1.f;
          lifted = true;
        }
      }
#pragma unroll
      for (int i = 0; i < RI; ++i) {
        const int head = rt * kKeyTile + 16 * r + mine + i;
        slope[r][i] = p.slopes != nullptr && head < p.group ? p.slopes[kv * p.group + head] * kLog2e : 0.f;
        m[r][i] = -__builtin_huge_valf();
        l[r][i] = 0.f;
        unit[r][i] = kMostUnit;
      }
#pragma unroll
      for (int i = 0; i < VB; ++i) o[r][i] = float4v{};
    }
    // Over the lanes that hold scores of the same row.
    auto across = [&](float x, auto&& with) {
#pragma unroll
      for (int i = 1; i < 64; i *= 2) {
        if (S::QP == 8 && i == 16) continue;
        if (S::QP == 16 && i >= 16) break;
        x = with(x, __shfl_xor(x, i));
      }
      return x;
    };

    __bf16* weights = reinterpret_cast<__bf16*>(keys + kKeys);
    float* factors = joint[0][wave];
    auto scale_sums = [&](int r) {  // by the rows' factors
      wave_order();
      const float f = factors[col % (RQ < 16 ? RQ : 16)];
      wave_order();
#pragma unroll
      for (int i = 0; i < VB; ++i) o[r][i] *= f;
    };
    for (; j0 < end; j0 += kStep) {
      // ---- scores ----
#pragma unroll
      for (int n = 0; n < NK; ++n) *reinterpret_cast<u32x4*>(keys + place_of(n * PER + lane / CH, lane % CH)) = k[n];
      wave_order();
      float w[NR][NS][4];
      float4v x[NR][4];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
#pragma unroll
        for (int r = 0; r < NR; ++r) x[r][s] = float4v{};
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
          const u32x4 piece = *reinterpret_cast<const u32x4*>(keys + place_of(16 * s + col, 4 * c + g));
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            x[r][s] = q[r][2 * c].template times<CODE>(u32x2{piece[0], piece[1]}, x[r][s]);
            x[r][s] = q[r][2 * c + 1].template times<CODE>(u32x2{piece[2], piece[3]}, x[r][s]);
          }
        }
      }
      wave_order();
#pragma unroll
      for (int r = 0; r < NR; ++r) {
#pragma unroll
        for (int i = 0; i < RI; ++i) {
          if constexpr (S::QP == 4) {
            w[r][0][i] = g < 2 ? (g == 0 ? x[r][0][i] : x[r][1][i]) : (g == 2 ? x[r][2][i] : x[r][3][i]);
          } else if constexpr (S::QP == 8) {
            w[r][0][i] = g < 2 ? x[r][0][i] : x[r][1][i];
            w[r][1][i] = g < 2 ? x[r][2][i] : x[r][3][i];
          } else {
#pragma unroll
            for (int s = 0; s < 4; ++s) w[r][s][i] = x[r][s][i];
          }
        }
      }
      float kscale[NS], vscale[NS];
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        kscale[s] = S::QP == 4 ? ks : __shfl(ks, key_of(s));
        vscale[s] = S::QP == 4 ? vs : __shfl(vs, key_of(s));
      }
      // ---- the next keys ----
      // (behind the last tile the rows of zeros again: under a condition all of the registers would be copied)
      find(j0 + kStep, next);
      load_k();
      next = page_of(j0 + 2 * kStep);
      // ---- weights ----
      const int left = end - j0;
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        // score = w * c + off (see Wave::weights)
        float c = sc.c, off = 0.f;
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int i = 0; i < RI; ++i) w[r][s][i] *= kscale[s];
        if constexpr (kUnits) {
          if (lifted) {
#pragma unroll
            for (int i = 0; i < RI; ++i)
#pragma unroll
              for (int s = 0; s < NS; ++s) w[r][s][i] *= shared.lifts[wave][16 * r + mine + i];
          }
        }
        if (sc.capped) {
          if (sizeof(T) == 2 && !sc.fine) {
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
              for (int i = 0; i < RI; ++i) w[r][s][i] = __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(w[r][s][i] * sc.inv2));
            c = 2.f * sc.cap;
            off = sc.cap;
          } else {
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
              for (int i = 0; i < RI; ++i) w[r][s][i] = tanh_of(w[r][s][i] * sc.inv);
            c = sc.cap;
          }
        }
        if (sc.biased) {
#pragma unroll
          for (int s = 0; s < NS; ++s) {
            const float away = static_cast<float>(len - 1 - j0 - key_of(s));
#pragma unroll
            for (int i = 0; i < RI; ++i) w[r][s][i] = fmaf(-slope[r][i], away, fmaf(w[r][s][i], c, off));
          }
          c = 1.f;
          off = 0.f;
        }
        if (left < kTile8) {
#pragma unroll
          for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int i = 0; i < RI; ++i)
              if (key_of(s) >= left) w[r][s][i] = -__builtin_huge_valf();
        }
        float top[RI];
        bool up = false, wide = false;
#pragma unroll
        for (int i = 0; i < RI; ++i) {
          top[i] = w[r][0][i];
#pragma unroll
          for (int s = 1; s < NS; ++s) top[i] = fmaxf(top[i], w[r][s][i]);
          top[i] = fmaf(top[i], c, off);
          up = up || top[i] > m[r][i] + kLag;
          wide = wide || fabsf(top[i]) > kWide;
        }
        if (__any(up)) {
#pragma unroll
          for (int i = 0; i < RI; ++i) {
            const float to = fmaxf(m[r][i], across(top[i], [](float x, float y) { return fmaxf(x, y); }));
            float f = to == m[r][i] ? 1.f : __builtin_amdgcn_exp2f(m[r][i] - to);
            m[r][i] = to;
            l[r][i] *= f;
            if constexpr (kUnits) {  // by the power of two that brings f to between 1/2 and 1
              const float by = fminf(__uint_as_float((253u - min(__float_as_uint(f) >> 23, 126u)) << 23), kMostUnit / unit[r][i]);
              unit[r][i] *= by;
              f *= by;
            }
            factors[mine + i] = f;  // (the same from all lanes of a row)
          }
          scale_sums(r);
        }
        const bool flat = __any(wide) != 0;  // (see kWide; nor would such a maximum hold kShift)
        if (flat) {
#pragma unroll
          for (int i = 0; i < RI; ++i)
#pragma unroll
            for (int s = 0; s < NS; ++s) w[r][s][i] = fmaf(w[r][s][i], c, off) - (m[r][i] == -__builtin_huge_valf() ? 0.f : m[r][i]);
          c = 1.f;
        }
        auto leave = [&](int s, int i, float rest) {  // the parts of a weight
          __bf16* to = weights + (16 * r + mine + i) * kRun8 + key_of(s);
          if (RQ >= 4 || mine == 0) {
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
              const __bf16 h = static_cast<__bf16>(rest);
              to[part * (R * kRun8)] = h;
              rest -= static_cast<float>(h);
            }
          }
        };
        bool far = false;
#pragma unroll
        for (int i = 0; i < RI; ++i) {
          const float ref = flat ? -kShift<T> : (m[r][i] == -__builtin_huge_valf() ? 0.f : m[r][i]) - kShift<T> - off;
#pragma unroll
          for (int s = 0; s < NS; ++s) {
            const float x = __builtin_amdgcn_exp2f(fmaf(w[r][s][i], c, -ref)) * kScale<T>;
            l[r][i] += x;
            if constexpr (kUnits) {
              w[r][s][i] = x;
              far = far || fabsf(x * unit[r][i] * vscale[s]) > 0x1p80f;
            } else {
              leave(s, i, x * vscale[s]);
            }
          }
        }
        if constexpr (kUnits) {
          if (__any(far)) {
#pragma unroll
            for (int i = 0; i < RI; ++i) {
              float most = 0.f;
#pragma unroll
              for (int s = 0; s < NS; ++s) most = fmaxf(most, w[r][s][i] * fabsf(vscale[s]));
              most = across(most, [](float x, float y) { return fmaxf(x, y); });
              float f = 1.f;
              if (most * unit[r][i] > 0x1p80f) {  // to 2^60 .. 2^61 (weights are at most 2^-16)
                const float to = __uint_as_float((314u - min(__float_as_uint(most) >> 23, 239u)) << 23);
                f = to / unit[r][i];
                unit[r][i] = to;
              }
              factors[mine + i] = f;
            }
            scale_sums(r);
          }
#pragma unroll
          for (int i = 0; i < RI; ++i)
#pragma unroll
            for (int s = 0; s < NS; ++s) leave(s, i, w[r][s][i] * unit[r][i] * vscale[s]);
        }
      }
      wave_order();
      // ---- sums ----
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        bhalf8 h[NR][PARTS];
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int part = 0; part < PARTS; ++part)
            h[r][part] = *reinterpret_cast<const bhalf8*>(weights + part * (R * kRun8) + (16 * r + col % (RQ < 16 ? RQ : 16)) * kRun8 + 32 * s + 8 * g);
#pragma unroll
        for (int i = 0; i < VB; ++i) {
          uint32_t x[8];
#pragma unroll
          for (int n8 = 0; n8 < 8; ++n8) x[n8] = v[s][n8][i >> 2];
          const bhalf8 a = bfloats_of_byte<CODE>(x, i & 3);
#pragma unroll
          for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int part = PARTS - 1; part >= 0; --part) o[r][i] = mma16(a, h[r][part], o[r][i]);
        }
      }
      wave_order();
      load_v();
    }

    // ---- join the four wavefronts: sums [wave][row][value] in LDS, then eight values a thread ----
    if constexpr (HEADS == 1) __syncthreads();  // (other wavefronts' weights have been read)
    float* so = reinterpret_cast<float*>(HEADS == 1 ? lds : keys);
    constexpr int kJoined = 4 / HEADS;
    const int part0 = HEADS == 1 ? 0 : wave, so_wave = HEADS == 1 ? wave : 0;
    if constexpr (kUnits) {  // out of their units
#pragma unroll
      for (int r = 0; r < NR; ++r) {
#pragma unroll
        for (int i = 0; i < RI; ++i) factors[mine + i] = 1.f / unit[r][i];
        scale_sums(r);
      }
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
#pragma unroll
      for (int i = 0; i < RI; ++i) {
        l[r][i] = across(l[r][i], [](float x, float y) { return x + y; });
        joint[0][wave][16 * r + mine + i] = m[r][i];
        joint[1][wave][16 * r + mine + i] = l[r][i];
      }
      if (col < RQ) {
#pragma unroll
        for (int n4 = 0; n4 < 4; ++n4)  // row 4 g + n4 of every block: values (4 g + n4) VB + {0 .. VB - 1}
#pragma unroll
          for (int i = 0; i < VB; i += 4)
            *reinterpret_cast<float4v*>(&so[(so_wave * R + 16 * r + col) * DP + (4 * g + n4) * VB + i]) =
                float4v{o[r][i][n4], o[r][i + 1][n4], o[r][i + 2][n4], o[r][i + 3][n4]};
      }
    }
    if constexpr (HEADS == 1) __syncthreads();
    else wave_order();
    Slot slot = {nullptr, orows};
    if (p.stiles > 0 || u0 > 0 || u1 < tiles)
      slot.at = p.part + e.first + ((static_cast<size_t>(at_slot) * p.otiles + rt) * p.hkv + kv) * slot_floats(orows, DP);
    for (int item = HEADS == 1 ? tid : lane; item < R * (DP / 8); item += kThreads / HEADS) {
      const int r = item / (DP / 8), d0 = item % (DP / 8) * 8, row = rt * kKeyTile + r;
      if (row >= p.group) break;
      float top = -__builtin_huge_valf(), f[kJoined], total = 0.f;
#pragma unroll
      for (int i = 0; i < kJoined; ++i) top = fmaxf(top, joint[0][part0 + i][r]);
#pragma unroll
      for (int i = 0; i < kJoined; ++i) {
        const float mi = joint[0][part0 + i][r];
        f[i] = mi == top ? 1.f : __builtin_amdgcn_exp2f(mi - top);
        total = fmaf(f[i], joint[1][part0 + i][r], total);
      }
      const float inv = slot.at != nullptr ? 1.f : inverse(total);
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = 0.f;
#pragma unroll
        for (int i = 0; i < kJoined; ++i) x[j] = fmaf(f[i], so[(i * R + r) * DP + d0 + j], x[j]);
        x[j] *= inv;
      }
      if (slot.at != nullptr) {
        float* to = slot.at + static_cast<size_t>(r) * DP + d0;
        *reinterpret_cast<float4v*>(to) = float4v{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<float4v*>(to + 4) = float4v{x[4], x[5], x[6], x[7]};
        if (d0 == 0) {
          slot_m<DP>(slot)[r] = top;
          slot_m<DP>(slot)[orows + r] = total;
        }
      } else if (d0 < p.d) {
        store_out<T, 8>(p.out + (static_cast<int64_t>(b) * p.hq + kv * p.group + row) * p.d * static_cast<int>(sizeof(T)), d0, x);
      }
    }
    todo -= u1 - u0;
    if (todo > 0) {
      len = uniform(length_of(p, ++b));
      u0 = 0;
      ++at_slot;
      ahead += tiles;
    } else {
      piece += e.shares;
      if (!has.pieces || !find_share(p, e, piece, has, deal)) break;
      b = has.seq;
      len = has.len;
      u0 = has.tile;
      todo = has.tiles;
      at_slot = has.slot;
      ahead = has.ahead;
    }
    if constexpr (HEADS == 1) __syncthreads();  // (the sums in LDS have been read)
    else wave_order();
  }
}

}  // namespace
}  // namespace g16
