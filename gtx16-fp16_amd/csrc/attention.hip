// Attention on the gfx950 matrix cores: prompts (g16_attention) and single tokens over a cache whose
// requests share a prefix (g16_attention_decode). The formulas and arguments stand in g16.h.
//
// Structure, for one key head and a tile of its query rows (row r of a sequence is token r / group,
// query head r % group: the query heads that share a key head share its tiles, too):
//   * Scores are computed transposed, S^T = K Q^T, in 32x32 blocks: a lane of the accumulator then holds
//     16 keys of ONE query row (lanes l and l + 32 the other half's), so a row's maximum and sum need one
//     exchange across the two halves, the running maximum, sum and rescale factor are one register each,
//     and the output is accumulated transposed as well, O^T += V^T P^T, each lane still on its own row.
//   * The weights P leave the score accumulator in exactly the order in which the next product wants
//     them: its 16-deep step s takes keys 16 s + 4 h + {0..3} and 16 s + 8 + 4 h + {0..3} from lane half h,
//     which are registers 8 s .. 8 s + 7 of the block. No weight moves between lanes. V^T comes from
//     row-major V in LDS in that order through the transposing reads (fp16) or plain dword reads (fp32).
//     fp16 inputs: each weight is rounded to fp16 for that product (its sum is not), which puts results 2.8e-4 from the
//     exact ones, where their own rounding to fp16 makes it 2.1e-4. Weights in two parts give 2.1e-4, and 8192 causal
//     tokens, 32 heads on 8 of 128, take 858 us instead of 633 (4 x 2048, 16 heads of 64: 73 and 58).
//   * One pass over the keys with a running maximum. A maximum only moves when a row's new one is more
//     than 2^kLag above it (the weights grow to at most 2^(kShift + kLag), far inside fp16), which after
//     the first tiles spares almost every rescale of O. fp16 weights are 2^kShift above their value,
//     which keeps those far below the maximum out of fp16's subnormals.
//   * fp32 values are multiplied as three bf16 parts each, v = hi + mid + lo: 8 bits a part, all 24 of the value, in
//     fp32's own range, so neither the size of a value nor that of its neighbours matters. Of the nine products of
//     parts the three below 2^-24 of the whole are left out; the other six take 192 cycles where eight
//     v_mfma_f32_32x32x2_f32 take 512 for the same step. Infinities have no parts (inf - inf), and the last parts of
//     values below 2^-110 are lost, which matters only beside huge ones: a tile of keys or values that holds one of
//     2^64 or more, or NaN, which every wavefront sees from the part it loaded, takes the fp32 instructions, and so do
//     all tiles of rows whose queries do. (32 x 256 tokens, 12 heads of 64, distance bias: 56 us; everything on the
//     fp32 instructions 71; two fp16 parts of 22 bits, right only for values of like size, 41.)
//   * Keys arrive by DMA into LDS with the row swizzles of Tile. A tile that ends past its sequence is cut
//     off by the buffer descriptor's range, which writes zeros: no value from behind a sequence's end
//     reaches a product.
// Two shapes of workgroup, both of 4 wavefronts:
//   * rows: 128 query rows, 32 per wavefront, all on the same keys, two tiles in LDS, one barrier a tile.
//   * keys: 32 query rows, every wavefront on its own tiles of 32 keys, joined at the end; for few rows, whose
//     time is that of one workgroup or of reading the keys.
// With too few tiles to fill the card, the keys are split over workgroups as well, which leave (O, maximum,
// sum) in the workspace (prompt_time weighs shapes and splits); a second launch joins them in split order (no
// atomics: repeated calls agree).
#include "attention8_own.hpp"

namespace g16 {
namespace {

using g16::uniform;

// Whether what a lane has seen is to be split: not where a value is 2^64 or more or not a number (or, which does no
// harm, where a sum of large ones is).
struct Range {
  float sum = 0.f;
  __device__ void see(float4v v) {
#pragma unroll
    for (int j = 0; j < 4; ++j) sum = fmaf(fabsf(v[j]), 0x1p64f, sum);
  }
  __device__ bool past() const { return __any(!(sum <= FLT_MAX)); }  // over the wavefront
};

// The value of the lane 32 away.
__device__ inline float other_half(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// One run of keys: the shared ones, or a sequence's own.
struct Keys {
  const char *k, *v;      // first key's row of this head
  uint32_t k_tok, v_tok;  // bytes between rows
  int len, pos0;          // keys; position of the first
};
struct KeyRuns {
  Keys shared, own;
  // (in scalar registers: the DMA's descriptors are made of them)
  __device__ Keys run(bool second) const {
    return Keys{uniform(second ? own.k : shared.k), uniform(second ? own.v : shared.v),
                static_cast<uint32_t>(uniform(static_cast<int>(second ? own.k_tok : shared.k_tok))),
                static_cast<uint32_t>(uniform(static_cast<int>(second ? own.v_tok : shared.v_tok))),
                uniform(second ? own.len : shared.len), uniform(second ? own.pos0 : shared.pos0)};
  }
};

template <typename V>
__device__ inline const __attribute__((address_space(3))) V* lds_at(uint32_t addr) {
  return reinterpret_cast<const __attribute__((address_space(3))) V*>(static_cast<uintptr_t>(addr));
}

// ---- tiles in LDS -------------------------------------------------------------------------------
// BN rows (keys) of DP values, 16-byte chunk c of row r at chunk position c ^ swizzle(r). K is read a
// row per lane (16 lanes cover 16 rows at one chunk: their positions differ in a 256-byte bank period);
// V in runs along a row, 4 rows and 64 bytes (fp16, transposing reads) or rows r and r + 4 and 128 bytes
// (fp32) at a time, which the swizzle puts on different banks.
template <typename T, int DP, int BN>
struct Tile {
  static constexpr int ROWB = DP * sizeof(T), RC = ROWB / 16, RPI = 64 / RC;
  static constexpr int BYTES = BN * ROWB, NI = BYTES / 1024;  // 1 KB DMA instructions
  using V8 = typename Vec8<T>::V;
  __device__ static int swz_k(int row) { return RC == 8 ? (row >> 1) & 7 : row & 15; }
  __device__ static int swz_v(int row) {
    if constexpr (sizeof(T) == 4) return ((row >> 2) & 1) << 3;
    else if constexpr (RC == 8) return (((row >> 1) & 1) << 2) | (((row >> 3) & 1) << 1);
    else return (row & 3) << 2;
  }
  // Within a row the swizzle and a step's chunks only touch different bits, so a lane's place in the tile
  // is one address per tile, and a step's an exclusive or and an immediate away from it.
  // K rows 32 kb + lane % 32 of the tile, values 16 ks + 8 (lane / 32) .. +7
  __device__ static uint32_t k_lane(int lane) {
    const int row = lane & 31, h = lane >> 5;
    return row * ROWB + (((sizeof(T) == 2 ? h : 2 * h) ^ swz_k(row)) << 4);
  }
  __device__ static V8 k_frag(uint32_t at, int kb, int ks) {
    if constexpr (sizeof(T) == 2) {
      return *lds_at<half8>((at ^ (ks * 32)) + kb * 32 * ROWB);
    } else {
      const float4v a = *lds_at<float4v>((at ^ (ks * 64)) + kb * 32 * ROWB);
      const float4v b = *lds_at<float4v>((at ^ (ks * 64 + 16)) + kb * 32 * ROWB);
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  // V^T row (value) 32 db + lane % 32, keys 16 ks + 4 h + {0..3} and 16 ks + 8 + 4 h + {0..3}
  __device__ static uint32_t v_lane(int lane) {
    const int h = lane >> 5, q = lane & 15;
    if constexpr (sizeof(T) == 2) {
      const int row = 4 * h + (q >> 2), chunk = 2 * ((lane >> 4) & 1) + ((q & 3) >> 1);
      return row * ROWB + ((chunk ^ swz_v(row)) << 4) + (q & 1) * 8;
    } else {
      const int row = 4 * h, chunk = (lane & 31) >> 2;
      return row * ROWB + ((chunk ^ swz_v(row)) << 4) + (lane & 3) * 4;
    }
  }
  __device__ static V8 v_frag(uint32_t at, int ks, int db) {
    if constexpr (sizeof(T) == 2) {
      half4 part[2];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const uint32_t x = at ^ (db * 64 + (swz_v(8 * g) << 4));
        part[g] = __builtin_bit_cast(half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds4_at(x + (16 * ks + 8 * g) * ROWB)));
      }
      return __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      float8v r;
#pragma unroll
      for (int j = 0; j < 8; ++j) r[j] = *lds_at<float>((at ^ (db * 128)) + (16 * ks + 8 * (j >> 2) + (j & 3)) * ROWB);
      return r;
    }
  }
};

// The byte offsets of a wavefront's DMA instructions first .. first + N - 1 within a tile of rows `tok`
// bytes apart: lane i's chunk of instruction n goes to LDS byte 1024 n + 16 i.
template <typename TL, int N, bool IS_V>
__device__ inline void dma_offsets(uint32_t (&off)[N], int first, int lane, uint32_t tok, int row_bytes) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int row = (first + n) * TL::RPI + lane / TL::RC;
    const int c = (lane % TL::RC) ^ (IS_V ? TL::swz_v(row) : TL::swz_k(row));
    off[n] = c * 16 < row_bytes ? static_cast<uint32_t>(row) * tok + c * 16 : kOob;
  }
}
template <int N>
__device__ inline void dma_rows(const char* base, uint32_t tok, int rows, const uint32_t (&off)[N], uint32_t lds) {
  const __amdgpu_buffer_rsrc_t r =
      __builtin_amdgcn_make_buffer_rsrc(uniform(const_cast<char*>(base)), 0, uniform(static_cast<int>(tok * static_cast<uint32_t>(rows))),
                                        kRawBufferDword3);
#pragma unroll
  for (int n = 0; n < N; ++n) dma16(r, lds + n * 1024, off[n]);
}
// The same from any address, for rows that lie in pages.
__device__ inline void dma16_from(const char* at, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds_addr)), "v"(at)
               : "memory", "m0");
}

// Where a wavefront takes a tile's operands from: LDS, or memory, where no other wavefront is needed (careful_rows).
template <typename TL>
struct InLds {
  uint32_t k_at, v_at;
  __device__ typename TL::V8 k(int kb, int ks) const { return TL::k_frag(k_at, kb, ks); }
  __device__ typename TL::V8 v(int ks, int db) const { return TL::v_frag(v_at, ks, db); }
};
template <typename T, int DP, int NB>
struct InMemory {
  const Keys& run;
  int j0, d, lane;
  using V8 = typename Vec8<T>::V;
  // (fp16 values are loaded as soon as the keys; fp32 ones would take too many registers)
  static constexpr bool HELD = sizeof(T) == 2;
  V8 held[HELD ? 2 * NB : 1][HELD ? DP / 32 : 1];
  __device__ InMemory(const Keys& r, int first, int values, int l) : run(r), j0(first), d(values), lane(l) {
    if constexpr (HELD) {
#pragma unroll
      for (int ks = 0; ks < 2 * NB; ++ks)
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) held[ks][db] = load(ks, db);
    }
  }
  __device__ V8 k(int kb, int ks) const {
    const int j = j0 + 32 * kb + (lane & 31), at = 16 * ks + 8 * (lane >> 5);
    // (Keys past the last one are the last one again: their weights are 0, and careful_rows takes the tile for one that
    // hides keys. Without a branch for each, a tile's loads are under way together.)
    const V8 x = *reinterpret_cast<const V8*>(run.k + static_cast<size_t>(min(j, run.len - 1)) * run.k_tok + min(at, d - 8) * sizeof(T));
    return at < d ? x : V8{};
  }
  __device__ V8 v(int ks, int db) const {
    if constexpr (HELD) return held[ks][db];
    else {
      asm volatile("" ::: "memory");
      return load(ks, db);
    }
  }
  __device__ V8 load(int ks, int db) const {
    const int at = 32 * db + (lane & 31), first = j0 + 16 * ks + 4 * (lane >> 5);
    V8 x = {};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = first + 8 * (i >> 2) + (i & 3);
      x[i] = *reinterpret_cast<const T*>(run.v + static_cast<size_t>(min(j, run.len - 1)) * run.v_tok + min(at, d - 1) * sizeof(T));
    }
    return x;
  }
};

// ---- one lane's query row ------------------------------------------------------------------------
struct Row {
  const char* q;  // NULL: no such row
  char* out;
  int pos, limit;  // position; last position it sees (INT_MAX: every key)
  float slope;     // slope * log2(e)
};

// What a workgroup needs to know besides its rows and keys.
struct What {
  Scoring sc;
  float sign;
  int d, causal;
};
__device__ inline What what_of(const Params& p) { return What{scoring(p), p.sign, p.d, p.causal}; }

__device__ inline float score_of(const Scoring& s, float x, float slope, float distance) {
  const float t = s.capped ? s.cap * tanh_of(x * s.inv) : x * s.c;
  return s.biased ? fmaf(-slope, fabsf(distance), t) : t;
}

// Of keys j0 .. j1 - 1 (at most 64), those with a value that is not finite.
template <typename T>
__device__ inline uint64_t infinite_keys(const Keys& run, int j0, int j1, int d, int lane) {
  using V8 = typename Vec8<T>::V;
  bool some = false;
  if (j0 + lane < j1) {
    const T* v = reinterpret_cast<const T*>(run.v + static_cast<size_t>(j0 + lane) * run.v_tok);
#pragma unroll 4
    for (int at = 0; at < d; at += 8) {
      const V8 x = *reinterpret_cast<const V8*>(v + at);
#pragma unroll
      for (int j = 0; j < 8; ++j) some |= !(fabsf(static_cast<float>(x[j])) <= FLT_MAX);
    }
  }
  return __ballot(some);
}

// ---- the running softmax and product of 32 rows in one wavefront ---------------------------------
template <typename T, int DP>
struct Wave {
  using V8 = typename Vec8<T>::V;
  decltype(operand(V8{})) q[DP / 16];
  float16v o[DP / 32];
  float m, l;  // the reference maximum (log2 units) and this lane's part of the sum of weights
  bool exact;  // fp32: whether a row of the wavefront is not to be split
  bool wide;   // whether a row's maximum is past kWide

  __device__ void start(const Row& row, float sign, int d, int lane) {
    const int h = lane >> 5;
    V8 v[DP / 16];
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      const int at = 16 * ks + 8 * h;
      v[ks] = V8{};
      if (row.q != nullptr && at < d) v[ks] = *reinterpret_cast<const V8*>(row.q + at * sizeof(T));
      if (sign != 1.f) v[ks] *= static_cast<T>(sign);
    }
    exact = false;
    if constexpr (sizeof(T) == 4) {
      Range r;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        r.see(__builtin_shufflevector(v[ks], v[ks], 0, 1, 2, 3));
        r.see(__builtin_shufflevector(v[ks], v[ks], 4, 5, 6, 7));
      }
      exact = r.past();
      if (__builtin_expect(exact, 0)) {
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) q[ks] = operand_of_any(v[ks]);
      }
    }
    if (!exact) {
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) q[ks] = operand(v[ks]);
    }
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) o[i] = float16v{};
    m = -__builtin_huge_valf();
    l = 0.f;
    wide = false;
  }

  // Keeps the sums whole up to here: taken apart for the stores below, they would be copied in every
  // pass of the loop before.
  __device__ void settle() {
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) asm volatile("" : "+v"(o[i]));
  }

  // S^T of the tile's NB blocks of 32 keys. EXACT: fp32 keys or queries that are not to be split (see Range).
  template <int NB, bool EXACT, bool FRESH, typename S>
  __device__ void products_as(const S& tile, float16v (&s)[NB]) const {
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
      s[kb] = float16v{};
      if constexpr (sizeof(T) == 4 && !EXACT) {
        // The small products first: each one added to the large ones' sum would round it (single tokens on 300 keys of
        // 64: 1.4e-7 from the exact result, 2.5e-7 a step at a time, in the same time).
        bhalf8 hi[DP / 16];
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          const Split8 key = operand(tile.k(kb, ks));
          s[kb] = mma_small(key, q[ks], s[kb]);
          hi[ks] = key.hi;
        }
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) s[kb] = mma(hi[ks], q[ks].hi, s[kb]);
      } else {
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          if constexpr (EXACT) {
            Split8 part = q[ks];
            // (or their sums would be kept in registers for the whole loop)
            if constexpr (FRESH) asm volatile("" : "+v"(part.hi), "+v"(part.mid), "+v"(part.lo));
            else asm volatile("" : "+v"(part.hi));
            s[kb] = mma(tile.k(kb, ks), whole(part), s[kb]);
          } else s[kb] = mma(tile.k(kb, ks), q[ks], s[kb]);
        }
      }
    }
  }
  // FRESH: the queries' parts are put together in every tile that needs them whole. Prompts are faster where only a part
  // of that is (32 x 256 tokens, 12 heads of 64: 59 us and 64), single tokens where all is (64 of 400 keys of 128 after
  // 8192: 147 and 150).
  template <int NB, bool FRESH, typename S>
  __device__ void products(const S& tile, float16v (&s)[NB], bool past) const {
    if constexpr (sizeof(T) == 4) {
      if (__builtin_expect(past || exact, 0)) {
        products_as<NB, true, FRESH>(tile, s);
        return;
      }
    }
    products_as<NB, false, FRESH>(tile, s);
  }

  // The weights of the tile's keys: positions pos0 .., `left` of them in the sequence.
  template <int NB>
  __device__ void weights(float16v (&s)[NB], const Scoring& sc, const Row& row, int pos0, int left, int last_seen, int lane) {
    const int h4 = (lane >> 5) * 4;
    // t = s * c + off
    float c = sc.c, off = 0.f;
    if (sc.capped) {
      if (sizeof(T) == 2 && !sc.fine) {
        // tanh(y) = 1 - 2 / (e^2y + 1): s becomes -1 / (e^2y + 1), and the rest of it joins c and off
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[kb][r] = __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(s[kb][r] * sc.inv2));
        c = 2.f * sc.cap;
        off = sc.cap;
      } else {
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[kb][r] = tanh_of(s[kb][r] * sc.inv);
        c = sc.cap;
      }
    }
    if (sc.biased) {
      const float at = static_cast<float>(row.pos - pos0 - h4);
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float e = static_cast<float>(32 * kb + 8 * (r >> 2) + (r & 3));
          s[kb][r] = fmaf(-row.slope, fabsf(at - e), fmaf(s[kb][r], c, off));
        }
      c = 1.f;
      off = 0.f;
    }
    if (left < 32 * NB || last_seen < pos0 + 32 * NB - 1) {
      const int lim = min(left - 1, row.limit - pos0) - h4;
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if (32 * kb + 8 * (r >> 2) + (r & 3) > lim) s[kb][r] = -__builtin_huge_valf();
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[kb][r]);
    top = fmaf(fmaxf(top, other_half(top)), c, off);
    // (-inf times c stays -inf: c > 0.) A lane whose maximum moves takes the whole wavefront along.
    if (__any(top > m + (wide ? 0.f : kLag))) {
      const float next = fmaxf(m, top);
      const float f = next == m ? 1.f : __builtin_amdgcn_exp2f(m - next);
      m = next;
      wide = __any(fabsf(next) > kWide && next != -__builtin_huge_valf()) != 0;
      l *= f;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] *= f;
    }
    // a row that has seen no key yet (m = -inf): every score is -inf, every weight 0
    const float from = m == -__builtin_huge_valf() ? 0.f : m;
    float ref = from - kShift<T> - off;
    if (wide) {  // (nor would such a maximum hold kShift, or a lag of kLag: fp16 weights would be infinite)
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[kb][r] = fmaf(s[kb][r], c, off) - from;
      c = 1.f;
      ref = -kShift<T>;
    }
    float sum = 0.f;
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float w = __builtin_amdgcn_exp2f(fmaf(s[kb][r], c, -ref)) * kScale<T>;
        s[kb][r] = w;
        sum += w;
      }
    l += sum;
  }

  template <int NB>
  __device__ static V8 weights_of(const float16v (&s)[NB], int ks) {
    V8 w;
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = static_cast<T>(s[ks >> 1][8 * (ks & 1) + j]);
    return w;
  }

  // O^T += V^T P^T. FINITE: without the values that are not.
  template <int NB, bool EXACT, bool FINITE, typename S>
  __device__ void add_as(const S& tile, const float16v (&s)[NB]) {
    auto values = [&](int ks, int db) {
      V8 v = tile.v(ks, db);
      if constexpr (FINITE) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!(fabsf(static_cast<float>(v[j])) <= FLT_MAX)) v[j] = static_cast<T>(0.f);
      }
      return v;
    };
#pragma unroll
    for (int ks = 0; ks < 2 * NB; ++ks) {
      const V8 w = weights_of(s, ks);
      if constexpr (EXACT) {
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) o[db] = mma(values(ks, db), w, o[db]);
      } else {
        const auto wp = operand(w);
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) o[db] = mma(operand(values(ks, db)), wp, o[db]);
      }
    }
  }
  // past: see Range. finite: without the tile's infinities and NaN.
  template <int NB, bool CAREFUL, typename S>
  __device__ void add(const S& tile, const float16v (&s)[NB], bool past, bool finite) {
    constexpr bool kF32 = sizeof(T) == 4;
    if constexpr (CAREFUL) {
      if (finite && (!kF32 || past)) {
        add_as<NB, kF32, true>(tile, s);
        return;
      }
    }
    if constexpr (kF32) {
      if (__builtin_expect(past, 0)) {
        add_as<NB, true, false>(tile, s);
        return;
      }
    }
    add_as<NB, false, false>(tile, s);
  }

  // Whether a sum of the wavefront's rows is not finite, other than of rows that are NaN by their weights already.
  __device__ bool infinite(const Row& row) const {
    float x = 0.f;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) x = fmaf(o[db][i], 0.f, x);
    return __any(x != 0.f && l == l && row.out != nullptr);
  }
  // The values of keys j0 .. j1 - 1 (at most 64) that are not finite, added for the rows that see them: their weights are
  // above 0, so that is what the product makes of them.
  __device__ void add_infinite(const Keys& run, int j0, int j1, const Row& row, int d, int lane) {
    for (uint64_t keys = infinite_keys<T>(run, j0, j1, d, lane); keys != 0; keys &= keys - 1) {
      const int j = j0 + __builtin_ctzll(keys);
      const T* v = reinterpret_cast<const T*>(run.v + static_cast<size_t>(j) * run.v_tok);
      const bool sees = run.pos0 + j <= row.limit && l == l;  // (with NaN weights, the row is NaN already)
      if (!__any(sees)) continue;
#pragma unroll
      for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int at = 32 * db + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
          const float x = at < d ? static_cast<float>(v[at]) : 0.f;
          if (sees && !(fabsf(x) <= FLT_MAX)) o[db][i] += x;
        }
    }
  }
};

// The rows of wavefront `wave` of a workgroup of 128 to their places.
template <typename T, int DP, int DU>
__device__ inline void store_rows(const Wave<T, DU>& w, const Row& row, int d, const Slot& slot, int wave, int lane) {
  const float l = w.l + other_half(w.l);
  const int h = lane >> 5, r = wave * 32 + (lane & 31);
  if (slot.at != nullptr) {
    float* o = slot.at + static_cast<size_t>(r) * DP;
#pragma unroll
    for (int db = 0; db < DU / 32; ++db)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float16v& a = w.o[db];
        *reinterpret_cast<float4v*>(o + 32 * db + 8 * q + 4 * h) = float4v{a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]};
      }
    if (h == 0) {
      slot_m<DP>(slot)[r] = w.m;
      slot_m<DP>(slot)[slot.rows + r] = l;
    }
  } else if (row.out != nullptr) {
    const float inv = inverse(l);
#pragma unroll
    for (int db = 0; db < DU / 32; ++db)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int d0 = 32 * db + 8 * q + 4 * h;
        const float v[4] = {w.o[db][4 * q] * inv, w.o[db][4 * q + 1] * inv, w.o[db][4 * q + 2] * inv, w.o[db][4 * q + 3] * inv};
        if (d0 < d) store_out<T, 4>(row.out, d0, v);
      }
  }
}

// (What arrives here is the same for all lanes, but for the row, and has to be known to be.)
__device__ inline What uniform(const What& c) {
  auto f = [](float x) { return __uint_as_float(static_cast<uint32_t>(uniform(static_cast<int>(__float_as_uint(x))))); };
  return What{{f(c.sc.c), f(c.sc.cap), f(c.sc.inv), f(c.sc.inv2), uniform(c.sc.capped) != 0, uniform(c.sc.fine) != 0, uniform(c.sc.biased) != 0},
              f(c.sign), uniform(c.d), uniform(c.causal)};
}

// A row's weight for a key that it does not see is 0, which times an infinity or NaN would be NaN. Hardly any value is one,
// so rows are computed as if none were. This computes those of a wavefront again whose sums are not finite, where such a
// value stands in a tile that hides keys from one of them (the last tiles): without these tiles' infinities and NaN,
// which are then added for the rows that see them. From memory: the workgroup's other wavefronts may have ended (waiting
// for them at the end of every call costs 48 documents of 200 tokens 5 %). 4096 tokens, 8 heads of 64 on 4: 55 us; with a
// NaN at key 40 66, at key 4086, for rows of which all keys are gone over again, 161; key by key and row by row it
// was 17 ms.
template <typename T, int DP, int DU>
__device__ __attribute__((noinline)) void careful_rows(What what, Row row, KeyRuns runs, int from0, int to0, int from1, int to1, int last, int limit,
                                                       Slot place) {
  constexpr int NB = sizeof(T) == 2 ? 2 : 1, BN = 32 * NB;
  const What c = uniform(what);
  const int last_seen = uniform(last), wave_limit = uniform(limit), lane = threadIdx.x & 63, wave = uniform(static_cast<int>(threadIdx.x >> 6));
  const Slot slot = {uniform(place.at), uniform(place.rows)};
  auto hides = [&](int first, int keys) { return keys < BN || last_seen < first + BN - 1; };
  auto tiles = [&](auto each) {  // of this wavefront, in order
    for (int g = 0; g < 2; ++g) {
      const Keys run = runs.run(g != 0);
      const int end = min(uniform(g ? to1 : to0), run.len);
      for (int j0 = uniform(g ? from1 : from0); j0 < end && run.pos0 + j0 <= wave_limit; j0 += BN) each(run, j0, run.pos0 + j0, run.len - j0);
    }
  };
  bool again = false;
  tiles([&](const Keys& run, int j0, int pos0, int left) {
    if (hides(pos0, left)) again = again || infinite_keys<T>(run, j0, min(j0 + BN, run.len), c.d, lane) != 0;
  });
  if (!again) return;
  Wave<T, DU> w;
  w.start(row, c.sign, c.d, lane);
  tiles([&](const Keys& run, int j0, int pos0, int left) {
    const InMemory<T, DU, NB> tile(run, j0, c.d, lane);
    float16v s[NB];
    w.template products_as<NB, sizeof(T) == 4, true>(tile, s);
    w.template weights<NB>(s, c.sc, row, pos0, left, last_seen, lane);
    if (hides(pos0, left)) w.template add_as<NB, sizeof(T) == 4, true>(tile, s);
    else w.template add_as<NB, sizeof(T) == 4, false>(tile, s);
  });
  tiles([&](const Keys& run, int j0, int pos0, int left) {
    if (hides(pos0, left)) w.add_infinite(run, j0, min(j0 + BN, run.len), row, c.d, lane);
  });
  store_rows<T, DP, DU>(w, row, c.d, slot, wave, lane);
}

// ---- workgroup of 128 rows ---------------------------------------------------------------------------
// Wavefront w holds rows 32 w .. 32 w + 31. last_seen: a position up to which every valid row of this
// wavefront sees; wave_limit: the last position that any of them sees. MASK: whether rows may not see keys. DU: of a row's DP places in LDS, those that
// the products go over, half of them for heads of up to 32 values, three quarters for up to 96 (8192 causal tokens, 32
// heads on 8 of 96: 483 us, all 128 places 569; 16 x 512 in fp32, 12 of 32: 64 and 95).
template <typename T, int DP, int DU, bool MASK, typename F>
__device__ inline void rows_workgroup(const Params& p, char* lds, int* ranges, const Row& row, const KeyRuns& runs, int n0, int tbeg, int tend,
                                      int last_seen, int wave_limit, const Slot& slot, const F& row_again) {
  constexpr int BN = sizeof(T) == 2 ? 64 : 32, NB = BN / 32;
  using TL = Tile<T, DP, BN>;
  constexpr int NIW = TL::NI / 4;  // DMA instructions of a wavefront per tile and operand
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const uint32_t base = lds_base(lds);
  const Scoring sc = scoring(p);
  uint32_t koff[NIW], voff[NIW];
  Keys at = {};  // the run, from the next tile to load on
  int pos0 = 0, left = 0, next_pos0, next_left;
  auto issue = [&](int t, int buf) {
    if (t == tbeg || t == n0) {  // a run begins
      at = runs.run(t >= n0);
      const int j0 = (t - (t >= n0 ? n0 : 0)) * BN;
      at.k += static_cast<size_t>(j0) * at.k_tok;
      at.v += static_cast<size_t>(j0) * at.v_tok;
      at.pos0 += j0;
      at.len -= j0;
      dma_offsets<TL, NIW, false>(koff, wave * NIW, lane, at.k_tok, p.d * static_cast<int>(sizeof(T)));
      dma_offsets<TL, NIW, true>(voff, wave * NIW, lane, at.v_tok, p.d * static_cast<int>(sizeof(T)));
    }
    const int rows = min(BN, at.len);
    const uint32_t to = base + buf * 2 * TL::BYTES + wave * NIW * 1024;
    dma_rows<NIW>(at.k, at.k_tok, rows, koff, to);
    dma_rows<NIW>(at.v, at.v_tok, rows, voff, to + TL::BYTES);
    next_pos0 = at.pos0;
    next_left = at.len;
    at.k += static_cast<size_t>(BN) * at.k_tok;
    at.v += static_cast<size_t>(BN) * at.v_tok;
    at.pos0 += BN;
    at.len -= BN;
  };
  Wave<T, DU> w;
  const uint32_t klane = base + TL::k_lane(lane), vlane = base + TL::BYTES + TL::v_lane(lane);
  if (tbeg < tend) issue(tbeg, 0);
  w.start(row, p.sign, p.d, lane);
  for (int t = tbeg; t < tend; ++t) {
    const uint32_t buf = static_cast<uint32_t>((t - tbeg) & 1);
    wait_dma_le<0>();
    if constexpr (sizeof(T) == 4) {  // the range of what this wavefront loaded, for all four
      Range k, v;
#pragma unroll
      for (int n = 0; n < NIW; ++n) {
        const uint32_t from = base + buf * 2 * TL::BYTES + (wave * NIW + n) * 1024 + lane * 16;
        k.see(*lds_at<float4v>(from));
        v.see(*lds_at<float4v>(from + TL::BYTES));
      }
      const int bits = (k.past() ? 1 : 0) | (v.past() ? 2 : 0);
      if (lane == 0) ranges[buf * 4 + wave] = bits;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    phase_barrier();  // tile t has arrived for every wavefront, and every one is done with tile t - 1
    int bits = 0;
    if constexpr (sizeof(T) == 4) bits = uniform(ranges[buf * 4] | ranges[buf * 4 + 1] | ranges[buf * 4 + 2] | ranges[buf * 4 + 3]);
    pos0 = next_pos0;
    left = next_left;
    if (t + 1 < tend) issue(t + 1, buf ^ 1);
    if (pos0 <= wave_limit) {
      float16v s[NB];
      const InLds<TL> tile = {klane + buf * 2 * TL::BYTES, vlane + buf * 2 * TL::BYTES};
      w.template products<NB, !MASK>(tile, s, (bits & 1) != 0);
      w.template weights<NB>(s, sc, row, pos0, left, last_seen, lane);
      w.template add<NB, false>(tile, s, (bits & 2) != 0, false);
    }
  }
  w.settle();
  store_rows<T, DP, DU>(w, row, p.d, slot, wave, lane);
  if constexpr (MASK) {
    if (p.causal && __builtin_expect(w.infinite(row), 0))
      careful_rows<T, DP, DU>(what_of(p), row_again(), runs, min(tbeg, n0) * BN, min(tend, n0) * BN, max(tbeg - n0, 0) * BN, max(tend - n0, 0) * BN,
                              last_seen, wave_limit, slot);
  }
}

// ---- workgroup of 32 rows, every wavefront on its own keys -------------------------------------------
// Wavefront w takes tiles tbeg + w, tbeg + w + 4, .. of 32 keys. K and V have one buffer each: the next K is on
// its way from the moment the scores are computed, the next V from that of the products, and a second
// workgroup on the CU fills the gaps (64 requests of up to 4096 keys, 8 key heads: 3.92 TB/s either way with
// two buffers each and one workgroup; 16 of up to 6000: 3.6, and 2.9 so).
// PAGED: the own keys may lie in pages. Of 16 keys or a multiple, as they mostly are, a page holds whole
// half tiles, whose pages are scalar loads a tile ahead; other sizes look up every key's page by itself.
struct Pages {
  const int32_t* table;  // this sequence's pages; NULL: its keys lie in a row
  int page, num_pages;
  int64_t k_seq, v_seq;
};
template <typename T, int DP>
__device__ void careful_keys(What c, char* lds, float* joint, Row row, KeyRuns runs, int n0, int tbeg, int tend, int last_seen, Slot slot);

// CAREFUL: as careful_rows, by the whole workgroup, whose wavefronts meet at the end anyway.
template <typename T, int DP, bool PAGED, bool MASK, bool CAREFUL = false>
__device__ inline void keys_workgroup(const What& c, char* lds, float* joint, const Row& row, const KeyRuns& runs, const Pages& pages,
                                      int n0, int tbeg, int tend, int last_seen, const Slot& slot) {
  constexpr int BN = 32;
  using TL = Tile<T, DP, BN>;
  constexpr int NI = TL::NI;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const uint32_t kl = lds_base(lds) + wave * (2 * TL::BYTES);  // K, then V
  const int row_bytes = c.d * static_cast<int>(sizeof(T));
  const bool paged = PAGED && pages.table != nullptr, whole = paged && pages.page % 16 == 0;
  uint32_t koff[NI], voff[NI];
  bool second = tbeg >= n0;  // the run that the offsets are for
  Keys cur = runs.run(second);
  auto offsets = [&]() {
    dma_offsets<TL, NI, false>(koff, 0, lane, cur.k_tok, row_bytes);
    dma_offsets<TL, NI, true>(voff, 0, lane, cur.v_tok, row_bytes);
  };
  offsets();
  // whole: the pages of a tile's two halves; else the page of this lane's key (lane % 32), in .x
  struct Ids {
    int x, y;
  };
  auto page_of = [&](int t) {
    Ids ids = {0, 0};
    if (!paged || t >= tend) return ids;
    const int j0 = (t - n0) * BN;
    if (whole) {
      // (constant address space: the table is only read, so these become scalar loads, which the waits for
      // the tiles do not count)
      auto* table = reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uint64_t>(pages.table));
      ids.x = table[j0 / pages.page];
      if (j0 + 16 < runs.own.len) ids.y = table[(j0 + 16) / pages.page];
    } else if (j0 + (lane & 31) < runs.own.len) {
      ids.x = pages.table[(j0 + (lane & 31)) / pages.page];
    }
    return ids;
  };
  auto dma_halves = [&](int j0, const Ids& ids, bool is_v, uint32_t to) {
    const char* base = is_v ? cur.v : cur.k;
    const uint32_t tok = is_v ? cur.v_tok : cur.k_tok;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int pg = g ? ids.y : ids.x, j = j0 + 16 * g;
      const bool known = static_cast<unsigned>(pg) < static_cast<unsigned>(pages.num_pages);
      const int rows = known ? max(0, min(16, cur.len - j)) : 0;
      const char* at = base + (known ? pg * (is_v ? pages.v_seq : pages.k_seq) + static_cast<int64_t>(j % pages.page) * tok : 0);
      const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(uniform(const_cast<char*>(at)), 0,
                                                                         uniform(static_cast<int>(tok * static_cast<uint32_t>(rows))), kRawBufferDword3);
#pragma unroll
      for (int n = 0; n < NI / 2; ++n) {
        const uint32_t off = is_v ? voff[g * (NI / 2) + n] : koff[g * (NI / 2) + n];
        // (an out-of-range offset stays one: less than 2^30 is taken off)
        dma16(r, to + (g * (NI / 2) + n) * 1024, off - 16 * g * tok);
      }
    }
  };
  auto dma_each = [&](int j0, int pg, bool is_v, uint32_t to) {
    const int j = j0 + (lane & 31);
    const char* at = nullptr;
    if (j < cur.len && static_cast<unsigned>(pg) < static_cast<unsigned>(pages.num_pages))
      at = (is_v ? cur.v : cur.k) + pg * (is_v ? pages.v_seq : pages.k_seq) +
           static_cast<int64_t>(j % pages.page) * (is_v ? cur.v_tok : cur.k_tok);
    const uint64_t a = reinterpret_cast<uint64_t>(at);
    const uint32_t lo = static_cast<uint32_t>(a), hi = static_cast<uint32_t>(a >> 32);
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      const int r = n * TL::RPI + lane / TL::RC;
      const int c = (lane % TL::RC) ^ (is_v ? TL::swz_v(r) : TL::swz_k(r));
      const uint64_t b = (static_cast<uint64_t>(static_cast<uint32_t>(__shfl(static_cast<int>(hi), r))) << 32) |
                         static_cast<uint32_t>(__shfl(static_cast<int>(lo), r));
      const char* from = b != 0 && c * 16 < row_bytes ? reinterpret_cast<const char*>(b) + c * 16
                                                      : reinterpret_cast<const char*>(g_zero_row);
      dma16_from(from, to + n * 1024);
    }
  };
  auto issue = [&](int t, const Ids& ids, bool is_v) {
    const uint32_t to = kl + (is_v ? TL::BYTES : 0);
    if (!second && t >= n0) {
      second = true;
      cur = runs.run(true);
      offsets();
    }
    const int j0 = (t - (second ? n0 : 0)) * BN;
    if (whole) {
      dma_halves(j0, ids, is_v, to);
    } else if (paged) {
      dma_each(j0, ids.x, is_v, to);
    } else {
      const int rows = min(BN, cur.len - j0);
      if (is_v) dma_rows<NI>(cur.v + static_cast<size_t>(j0) * cur.v_tok, cur.v_tok, rows, voff, to);
      else dma_rows<NI>(cur.k + static_cast<size_t>(j0) * cur.k_tok, cur.k_tok, rows, koff, to);
    }
  };
  const InLds<TL> tile = {kl + TL::k_lane(lane), kl + TL::BYTES + TL::v_lane(lane)};
  auto past = [&](uint32_t tile) {
    if constexpr (sizeof(T) == 2) return false;
    Range r;
#pragma unroll
    for (int n = 0; n < NI; ++n) r.see(*lds_at<float4v>(tile + n * 1024 + lane * 16));
    return r.past();
  };
  Wave<T, DP> w;
  auto hides = [&](int first, int keys) { return last_seen < first + min(keys, BN) - 1; };
  // this wavefront's tiles that hide keys, from the last one on
  auto hidden = [&](auto each) {
    for (int u = tend - 1; u >= tbeg; --u) {
      const Keys run = runs.run(u >= n0);
      const int j0 = (u - (u >= n0 ? n0 : 0)) * BN;
      if (!hides(run.pos0 + j0, run.len - j0)) break;
      if ((u - tbeg) % 4 == wave) each(run, j0, min(j0 + BN, run.len));
    }
  };
  int t = tbeg + wave;
  if (t < tend) {
    const Ids ids = page_of(t);
    issue(t, ids, false);
    issue(t, ids, true);
  }
  Ids next = page_of(t + 4);
  w.start(row, c.sign, c.d, lane);
  // The rows' loads are done before the loop: its waits count DMA only, and the compiler, which does not
  // know of that, would wait for all of it before it first uses the rows.
  __builtin_amdgcn_s_waitcnt(0);
  for (; t < tend; t += 4) {
    const bool more = t + 4 < tend, own = t >= n0;
    const int j0 = (t - (own ? n0 : 0)) * BN;
    const int pos0 = (own ? runs.own.pos0 : runs.shared.pos0) + j0, left = (own ? runs.own.len : runs.shared.len) - j0;
    float16v s[1];
    // Waits for K, then for V: only the instructions issued after it may be in flight (others among them only
    // make it wait longer).
    wait_dma_le<NI>();
    w.template products<1, !MASK>(tile, s, past(kl));
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K has been read before the next K overwrites it
    if (more) issue(t + 4, next, false);
    w.template weights<1>(s, c.sc, row, pos0, left, last_seen, lane);
    if (more) wait_dma_le<NI>();
    else wait_dma_le<0>();
    w.template add<1, CAREFUL>(tile, s, past(kl + TL::BYTES), CAREFUL && hides(pos0, left));
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (more) issue(t + 4, next, true);
    next = page_of(t + 8);
  }
  w.settle();
  if constexpr (CAREFUL) hidden([&](const Keys& run, int j0, int j1) { w.add_infinite(run, j0, j1, row, c.d, lane); });
  // ---- join the four wavefronts: sums [wave][value][row] in LDS, then 8 threads a row ----
  const float l = w.l + other_half(w.l);
  const int h = lane >> 5, r = lane & 31;
  __syncthreads();
  float* so = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) so[(wave * DP + 32 * db + 8 * (i >> 2) + 4 * h + (i & 3)) * 32 + r] = w.o[db][i];
  if (h == 0) {
    joint[wave * 32 + r] = w.m;
    joint[128 + wave * 32 + r] = l;
  }
  if (MASK && tid < 2) joint[256 + tid] = 0.f;
  __syncthreads();
  float top = -__builtin_huge_valf();
#pragma unroll
  for (int i = 0; i < 4; ++i) top = fmaxf(top, joint[i * 32 + r]);
  float f[4], total = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float mi = joint[i * 32 + r];
    f[i] = mi == top ? 1.f : __builtin_amdgcn_exp2f(mi - top);
    total += f[i] * joint[128 + i * 32 + r];
  }
  constexpr int DT = DP / 8;  // values a thread: d0 .. d0 + DT - 1
  const int d0 = (tid >> 5) * DT;
  const float inv = slot.at != nullptr ? 1.f : inverse(total);
  float bad = 0.f;
  const bool stored = slot.at != nullptr ? r < slot.rows : row.out != nullptr;
#pragma unroll
  for (int e0 = 0; e0 < DT; e0 += 8) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float x = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) x = fmaf(f[i], so[(i * DP + d0 + e0 + e) * 32 + r], x);
      v[e] = x * inv;
      bad = fmaf(x, 0.f, bad);
    }
    if (stored && slot.at != nullptr) {
      float* o = slot.at + static_cast<size_t>(r) * DP + d0 + e0;
      *reinterpret_cast<float4v*>(o) = float4v{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<float4v*>(o + 4) = float4v{v[4], v[5], v[6], v[7]};
    } else if (stored && d0 + e0 < c.d) {
      store_out<T, 8>(row.out, d0 + e0, v);
    }
  }
  if (slot.at != nullptr && tid < 32 && r < slot.rows) {
    slot_m<DP>(slot)[r] = top;
    slot_m<DP>(slot)[slot.rows + r] = total;
  }
  if constexpr (MASK && !CAREFUL) {
    if (!c.causal) return;
    // whether sums are not finite, then whether hidden values are
    uint32_t* flags = reinterpret_cast<uint32_t*>(joint + 256);
    if (__any(bad != 0.f && total == total && row.q != nullptr) && lane == 0) atomicOr(flags, 1u);
    __syncthreads();
    if (__builtin_expect(uniform(static_cast<int>(flags[0])), 0)) {
      hidden([&](const Keys& run, int j0, int j1) {
        if (infinite_keys<T>(run, j0, j1, c.d, lane) != 0 && lane == 0) atomicOr(flags + 1, 1u);
      });
      __syncthreads();
      if (uniform(static_cast<int>(flags[1]))) careful_keys<T, DP>(c, lds, joint, row, runs, n0, tbeg, tend, last_seen, slot);
    }
  }
}
template <typename T, int DP>
__device__ __attribute__((noinline)) void careful_keys(What c, char* lds, float* joint, Row row, KeyRuns runs, int n0, int tbeg, int tend, int last_seen,
                                                       Slot slot) {
  keys_workgroup<T, DP, false, true, true>(uniform(c), uniform(lds), uniform(joint), row, runs, Pages{}, uniform(n0), uniform(tbeg), uniform(tend),
                                           uniform(last_seen), Slot{uniform(slot.at), uniform(slot.rows)});
}

template <typename T, int DP>
constexpr int rows_lds() {
  return 4 * Tile<T, DP, sizeof(T) == 2 ? 64 : 32>::BYTES;
}
constexpr int cmax(int a, int b) { return a > b ? a : b; }
template <typename T, int DP>
constexpr int keys_lds() {
  return cmax(8 * Tile<T, DP, 32>::BYTES, 4 * DP * 32 * 4);  // (the second: joining the wavefronts)
}

// ---- prompts -------------------------------------------------------------------------------------------
// Row tile t of all sequences' tiles of `rt` rows: its sequence and where that sequence's rows and keys
// are. Packed sequences: every wavefront counts the tiles of 64 sequences at a time. false: past the end.
struct Where {
  int seq, tile, lq, lk;
  int64_t q0, k0;  // first row, first key (packed)
};
__device__ inline bool find_tile(const Params& p, int t, int rt, Where& w) {
  if (p.q_off == nullptr) {
    // equal sequences: the last tiles first (under a causal mask they have the most keys)
    w.lq = p.q_len;
    w.lk = p.k_len;
    const int each = ceil_div(p.q_len * p.group, rt);
    w.seq = t % p.seqs;
    w.tile = each - 1 - t / p.seqs;
    w.q0 = w.k0 = 0;
    return w.tile >= 0;
  }
  const int lane = threadIdx.x & 63;
  for (int b0 = 0; b0 < p.seqs; b0 += kWave) {
    const int b = b0 + lane;
    int q0 = 0, lq = 0, k0 = 0, lk = 0;
    if (b < p.seqs) {  // (all four loads together: one round trip before the keys)
      const int qa = p.q_off[b], qb = p.q_off[b + 1], ka = p.k_off[b], kb = p.k_off[b + 1];
      q0 = min(max(qa, 0), p.q_len);
      lq = max(min(qb, p.q_len) - q0, 0);
      k0 = min(max(ka, 0), p.k_len);
      lk = max(min(kb, p.k_len) - k0, 0);
    }
    const int n = static_cast<int>((static_cast<int64_t>(lq) * p.group + rt - 1) / rt);
    int upto = n;
#pragma unroll
    for (int i = 1; i < kWave; i *= 2) {
      const int x = __shfl_up(upto, i);
      if (lane >= i) upto += x;
    }
    const uint64_t hit = __ballot(t < upto);
    if (hit != 0) {
      const int l = __builtin_ctzll(hit);
      w.seq = b0 + l;
      w.lq = __builtin_amdgcn_readlane(lq, l);
      w.lk = __builtin_amdgcn_readlane(lk, l);
      w.q0 = __builtin_amdgcn_readlane(q0, l);
      w.k0 = __builtin_amdgcn_readlane(k0, l);
      w.tile = __builtin_amdgcn_readlane(upto, l) - 1 - t;  // the sequence's last tile first
      return true;
    }
    t -= __builtin_amdgcn_readlane(upto, kWave - 1);
  }
  return false;
}

// A row of the sequence `w`.
__device__ inline Row prompt_row(const Params& p, const Where& w, int kv, int r, int size) {
  Row row;
  const int tok = r / p.group, head = kv * p.group + r % p.group;
  const bool ok = tok < w.lq;
  const int64_t at = (p.q_off == nullptr ? static_cast<int64_t>(w.seq) * p.q_len : w.q0) + tok;
  row.q = ok ? p.q + (p.q_off == nullptr ? w.seq * p.q_seq : w.q0 * p.q_tok) + tok * p.q_tok + head * p.q_head : nullptr;
  row.out = ok ? p.out + (at * p.hq + head) * p.d * size : nullptr;
  row.pos = p.shared + w.lk - w.lq + tok;
  row.limit = p.causal ? max(row.pos, p.visible != nullptr ? max(p.visible[w.seq], 0) - 1 : -1) : 0x7fffffff;
  row.slope = p.slopes != nullptr && ok ? p.slopes[head] * kLog2e : 0.f;
  return row;
}

// (three workgroups of 128 rows fit a CU at 64 values a row, two at 128)
template <typename T, int DP, int DU, bool KEYS>
__global__ __launch_bounds__(kThreads, DP == 64 && (!KEYS || sizeof(T) == 2) ? 3 : 2) void prompt_kernel(Params p) {
  constexpr int RT = KEYS ? kKeyTile : kRowTile, BN = KEYS ? 32 : (sizeof(T) == 2 ? 64 : 32);
  __shared__ __attribute__((aligned(1024))) char lds[KEYS ? keys_lds<T, DP>() : rows_lds<T, DP>()];
  __shared__ float joint[KEYS ? 258 : 1];
  __shared__ int ranges[8];  // fp32: of the two tiles in LDS, from each wavefront
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  int lin = blockIdx.x;
  const int kv = lin % p.hkv;
  lin /= p.hkv;
  const int split = lin % p.splits, t = lin / p.splits;
  Where w;
  if (!find_tile(p, t, RT, w)) return;
  const int r0 = w.tile * RT, first = r0 + (KEYS ? 0 : 32 * wave);
  const Row row = prompt_row(p, w, kv, first + (lane & 31), sizeof(T));
  const KeyRuns runs = {
      {p.sk + kv * p.sk_head, p.sv + kv * p.sv_head, p.sk_tok, p.sv_tok, p.shared, 0},
      {p.k + (p.k_off == nullptr ? w.seq * p.k_seq : w.k0 * p.k_tok) + kv * p.k_head,
       p.v + (p.k_off == nullptr ? w.seq * p.v_seq : w.k0 * p.v_tok) + kv * p.v_head, p.k_tok, p.v_tok, w.lk, p.shared}};
  // the keys that some row of the tile sees
  int seen = 0x7fffffff, last_seen = 0x7fffffff, wave_limit = 0x7fffffff;
  if (p.causal) {
    const int vis = p.visible != nullptr ? max(uniform(p.visible[w.seq]), 0) - 1 : -1;
    const int pos0 = p.shared + w.lk - w.lq;
    const int last_tok = min(r0 + RT - 1, w.lq * p.group - 1) / p.group;
    seen = max(pos0 + last_tok, vis);
    last_seen = max(pos0 + first / p.group, vis);
    wave_limit = max(pos0 + min(first + 31, w.lq * p.group - 1) / p.group, vis);
  }
  if (first >= w.lq * p.group) wave_limit = -1;  // no such rows
  const int end0 = min(p.shared, seen < 0 ? 0 : (seen == 0x7fffffff ? seen : seen + 1));
  const int end1 = min(w.lk, seen < p.shared ? 0 : (seen == 0x7fffffff ? seen : seen + 1 - p.shared));
  const int n0 = ceil_div(end0, BN), n = n0 + ceil_div(end1, BN);
  const int tbeg = share_begin(n, split, p.splits), tend = share_begin(n, split + 1, p.splits);
  Slot slot = {nullptr, RT};
  if (p.splits > 1) slot.at = p.part + static_cast<size_t>(blockIdx.x) * slot_floats(RT, DP);
  if constexpr (KEYS) {
    keys_workgroup<T, DP, false, true>(what_of(p), lds, joint, row, runs, Pages{}, n0, tbeg, tend, last_seen, slot);
  } else {
    rows_workgroup<T, DP, DU, true>(p, lds, ranges, row, runs, n0, tbeg, tend, last_seen, wave_limit, slot,
                                    [&]() { return prompt_row(p, w, kv, first + (lane & 31), sizeof(T)); });
  }
}

constexpr int kJoinRows = 8;  // rows of a workgroup of the joining kernels: two a wavefront

template <typename T, int DP>
__global__ __launch_bounds__(kThreads) void prompt_join_kernel(Params p, int rt) {
  const int per = rt / kJoinRows, wave = uniform(threadIdx.x >> 6);
  const int chunk = blockIdx.x % per, lin = blockIdx.x / per;
  const int kv = lin % p.hkv, t = lin / p.hkv;
  Where w;
  if (!find_tile(p, t, rt, w)) return;
  for (int i = 0; i < kJoinRows / 4; ++i) {
    const int r = chunk * kJoinRows + i * 4 + wave;
    const int tok = (w.tile * rt + r) / p.group, head = kv * p.group + (w.tile * rt + r) % p.group;
    if (tok >= w.lq) break;
    const int64_t at = (p.q_off == nullptr ? static_cast<int64_t>(w.seq) * p.q_len : w.q0) + tok;
    join_row<T, DP>(p.out + (at * p.hq + head) * p.d * static_cast<int>(sizeof(T)), p.d, p.splits,
                    [&](int s, const float*& o, const float*& m, int& rows) {
                      const float* slot = p.part + (static_cast<size_t>(t * p.splits + s) * p.hkv + kv) * slot_floats(rt, DP);
                      o = slot + static_cast<size_t>(r) * DP;
                      m = slot + static_cast<size_t>(rt) * DP + r;
                      rows = rt;
                    });
  }
}

// ---- single tokens -------------------------------------------------------------------------------------
// Workgroups [0, stiles * ssplits * hkv): the shared keys, for the rows (request, query head) of all
// requests at once. Then the requests' own keys, 32 rows a tile, in parts of about equal length over all
// requests: the device knows their lengths, so every wavefront adds them up and finds its part (see Part).
// Slots in the same order. A request's only part writes the output itself.
__device__ inline Row token_row(const Params& p, int b, int head, bool ok, int size) {
  Row row;
  row.q = ok ? p.q + b * p.q_seq + head * p.q_head : nullptr;
  row.out = ok ? p.out + (static_cast<int64_t>(b) * p.hq + head) * p.d * size : nullptr;
  const int len = ok ? length_of(p, b) : 0;
  row.pos = p.shared + len - 1;
  row.limit = 0x7fffffff;
  row.slope = ok && p.slopes != nullptr ? p.slopes[head] * kLog2e : 0.f;
  return row;
}

// Workgroup `block` of those for the shared keys. ranges: 8 values in LDS, where workgroups have 128 rows.
template <typename T, int DP, bool SKEYS>
__device__ inline void shared_workgroup(const Params& p, int block, char* lds, float* joint, int* ranges) {
  constexpr int SRT = SKEYS ? kKeyTile : kRowTile, SBN = SKEYS ? 32 : (sizeof(T) == 2 ? 64 : 32);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  int lin = block;
  const int kv = lin % p.hkv;
  lin /= p.hkv;
  // (a split's row tiles next to each other: they read the same keys)
  const int t = lin % p.stiles, split = lin / p.stiles;
  const int r = t * SRT + (SKEYS ? 0 : 32 * wave) + (lane & 31);
  const int b = r / p.group;
  const Row row = token_row(p, b, kv * p.group + r % p.group, b < p.seqs, sizeof(T));
  const KeyRuns runs = {{p.sk + kv * p.sk_head, p.sv + kv * p.sv_head, p.sk_tok, p.sv_tok, p.shared, 0}, {}};
  const int n = ceil_div(p.shared, SBN);
  const int tbeg = share_begin(n, split, p.ssplits), tend = share_begin(n, split + 1, p.ssplits);
  Slot slot = {p.part + (static_cast<size_t>(t * p.ssplits + split) * p.hkv + kv) * slot_floats(SRT, DP), SRT};
  if constexpr (SKEYS) {
    keys_workgroup<T, DP, false, false>(what_of(p), lds, joint, row, runs, Pages{}, n, tbeg, tend, 0x7fffffff, slot);
  } else {
    const bool some = t * SRT + 32 * wave < p.seqs * p.group;  // a wavefront without rows computes nothing
    rows_workgroup<T, DP, DP, false>(p, lds, ranges, row, runs, n, tbeg, tend, 0x7fffffff, some ? 0x7fffffff : -1, slot, [&]() { return row; });
  }
}

template <typename T, int DP, bool SKEYS>
__global__ __launch_bounds__(kThreads, 2) void decode_kernel(Params p) {
  constexpr int SRT = SKEYS ? kKeyTile : kRowTile;
  __shared__ __attribute__((aligned(1024))) char lds[SKEYS ? keys_lds<T, DP>() : cmax(keys_lds<T, DP>(), rows_lds<T, DP>())];
  __shared__ float joint[256];
  __shared__ int ranges[8];
  const int lane = threadIdx.x & 63;
  const int nshared = p.stiles * p.ssplits * p.hkv;
  if (static_cast<int>(blockIdx.x) < nshared) {
    shared_workgroup<T, DP, SKEYS>(p, static_cast<int>(blockIdx.x), lds, joint, ranges);
    return;
  }
  int lin = blockIdx.x - nshared;
  const int own = lin;
  const int kv = lin % p.hkv;
  lin /= p.hkv;
  const int rt = lin % p.otiles;
  Part part;
  if (!find_part(p, lin / p.otiles, true, part)) return;
  const int b = part.seq, len = part.len;
  const int orows = own_rows(p.group), r = rt * kKeyTile + (lane & 31);
  const Row row = token_row(p, b, kv * p.group + r, r < p.group, sizeof(T));
  KeyRuns runs = {{}, {p.k + kv * p.k_head, p.v + kv * p.v_head, p.k_tok, p.v_tok, len, p.shared}};
  const Pages pages = {p.pages == nullptr ? nullptr : p.pages + static_cast<size_t>(b) * p.max_pages, p.page, p.num_pages, p.k_seq, p.v_seq};
  if (p.pages == nullptr) {
    runs.own.k += b * p.k_seq;
    runs.own.v += b * p.v_seq;
  }
  const int n = ceil_div(len, 32);
  const int tbeg = share_begin(n, part.split, part.splits), tend = share_begin(n, part.split + 1, part.splits);
  Slot slot = {nullptr, orows};
  if (p.stiles > 0 || part.splits > 1) slot.at = p.part + static_cast<size_t>(nshared) * slot_floats(SRT, DP) + static_cast<size_t>(own) * slot_floats(orows, DP);
  keys_workgroup<T, DP, true, false>(what_of(p), lds, joint, row, runs, pages, 0, tbeg, tend, 0x7fffffff, slot);
}

// The shared keys for few rows and, over a cache of 8 bits, the own ones in one launch: one after the other, each would leave the
// card half empty (16 requests of up to 1500 in int8 after 2048, 32 heads on 8 of 128, in a graph: 31.6 us, so 22.4).
template <int DP, int CODE, int RQ, int HEADS>
__global__ __launch_bounds__(kThreads, 2) void decode_both8_kernel(Params p, Params8 e) {
  __shared__ union Lds {
    Lds8<_Float16, DP, RQ> own;
    struct {
      alignas(1024) char tiles[keys_lds<_Float16, DP>()];
      float joint[256];
    } shared;
  } lds;
  const int nshared = p.stiles * p.ssplits * p.hkv;
  if (static_cast<int>(blockIdx.x) < nshared) shared_workgroup<_Float16, DP, true>(p, static_cast<int>(blockIdx.x), lds.shared.tiles, lds.shared.joint, nullptr);
  else own8_workgroup<_Float16, DP, CODE, RQ, true, HEADS>(p, e, static_cast<int>(blockIdx.x) - nshared, lds.own);
}

template <typename T, int DP>
__global__ __launch_bounds__(kThreads) void decode_join_kernel(Params p, int srt) {
  const int row = uniform(static_cast<int>(blockIdx.x) * 4 + static_cast<int>(threadIdx.x >> 6));
  if (row >= p.seqs * p.hq) return;
  const int b = row / p.hq, head = row % p.hq, kv = head / p.group, g = head % p.group;
  const int ns = p.stiles > 0 ? p.ssplits : 0, orows = own_rows(p.group);
  const size_t nshared = static_cast<size_t>(p.stiles) * p.ssplits * p.hkv;
  const int sr = b * p.group + g;
  Part part;
  if (!find_part(p, b, false, part) || ns + part.splits == 1) return;
  join_row<T, DP>(p.out + static_cast<int64_t>(row) * p.d * static_cast<int>(sizeof(T)), p.d, ns + part.splits,
                  [&](int i, const float*& o, const float*& m, int& rows) {
                    const float* slot;
                    int r;
                    if (i < ns) {
                      slot = p.part + (static_cast<size_t>((sr / srt) * p.ssplits + i) * p.hkv + kv) * slot_floats(srt, DP);
                      r = sr % srt;
                      rows = srt;
                    } else {
                      const size_t at = (static_cast<size_t>(part.first + i - ns) * p.otiles + g / kKeyTile) * p.hkv + kv;
                      slot = p.part + nshared * slot_floats(srt, DP) + at * slot_floats(orows, DP);
                      r = g % kKeyTile;
                      rows = orows;
                    }
                    o = slot + static_cast<size_t>(r) * DP;
                    m = slot + static_cast<size_t>(rows) * DP + r;
                  });
}

// ---- host ------------------------------------------------------------------------------------------------

// (what the Python binding packs)
static_assert(sizeof(g16_attention_args) == 12 * 8 + 13 * 8 + 16 * 4 + 16, "no padding");

int cus_of(const g16_attention_args& a) {
  if (a.num_cus > 0) return a.num_cus;
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return 256;
  return n > 0 ? n : 256;
}

// What the entry points check; the strides of operands without elements are not looked at. codes: the cache is in 8 bits,
// whose rows are read by addresses of their own.
int check(const g16_attention_args& a, bool decode, bool codes = false) {
  const int size = a.is_f32 ? 4 : 2;
  if (a.is_f32 != 0 && a.is_f32 != 1) return G16_E_DTYPE;
  if (a.seqs < 0 || a.q_len < 0 || a.k_len < 0 || a.hq < 0 || a.hkv < 0 || a.shared < 0 || a.d <= 0 || a.d % 8 != 0 ||
      a.d > G16_ATTENTION_MAX_D)
    return G16_E_SHAPE;
  if (a.seqs == 0 || a.hq == 0 || (!decode && a.q_len == 0)) return G16_OK;
  if (a.hkv == 0 || a.hq % a.hkv != 0 || !(a.softcap >= 0.f && a.softcap <= FLT_MAX) || !(a.scale == a.scale)) return G16_E_SHAPE;
  if (static_cast<int64_t>(a.shared) + a.k_len > (1 << 30) || static_cast<int64_t>(a.q_len) * a.hq > (1LL << 31) - 1 ||
      static_cast<int64_t>(a.seqs) * a.hq > (1LL << 31) - 1)
    return G16_E_SHAPE;
  if (a.q == nullptr || a.out == nullptr) return G16_E_NULL;
  auto row = [&](int64_t token, int64_t head, bool longest) {
    const int64_t t = token * size, h = head * size;
    return t % 16 == 0 && h % 16 == 0 && (!longest || (token >= a.d && t < G16_ATTENTION_MAX_STRIDE));
  };
  if (!aligned16(a.q) || !aligned16(a.out) || !row(decode ? 0 : a.q_token, a.q_head, false) || a.q_seq * size % 16 != 0) return G16_E_ALIGN;
  if (a.k_len > 0) {
    if (a.k == nullptr || a.v == nullptr) return G16_E_NULL;
    if (codes) {
      const int64_t all = a.k_seq | a.k_token | a.k_head | a.v_seq | a.v_token | a.v_head | static_cast<int64_t>(reinterpret_cast<uintptr_t>(a.k)) |
                          static_cast<int64_t>(reinterpret_cast<uintptr_t>(a.v));
      if (all % 8 != 0) return G16_E_ALIGN;
    } else if (!aligned16(a.k) || !aligned16(a.v) || a.k_seq * size % 16 != 0 || a.v_seq * size % 16 != 0) {
      return G16_E_ALIGN;
    } else if (!row(a.k_token, a.k_head, true) || !row(a.v_token, a.v_head, true)) {
      return G16_E_SHAPE;
    }
  }
  if (a.shared > 0) {
    if (a.shared_k == nullptr || a.shared_v == nullptr) return G16_E_NULL;
    if (!aligned16(a.shared_k) || !aligned16(a.shared_v)) return G16_E_ALIGN;
    if (!row(a.shared_k_token, a.shared_k_head, true) || !row(a.shared_v_token, a.shared_v_head, true)) return G16_E_SHAPE;
  }
  if (decode) {
    if (a.lengths == nullptr) return G16_E_NULL;
    if (a.page < 0 || a.max_pages < 0 || a.num_pages < 0) return G16_E_SHAPE;
    if (a.pages != nullptr && (a.page <= 0 || static_cast<int64_t>(a.page) * a.max_pages < a.k_len)) return G16_E_SHAPE;
  } else if ((a.q_offsets == nullptr) != (a.k_offsets == nullptr)) {
    return G16_E_NULL;
  }
  return G16_OK;
}

Params params(const g16_attention_args& a) {
  const int64_t size = a.is_f32 ? 4 : 2;
  Params p = {};
  p.q = static_cast<const char*>(a.q);
  p.k = static_cast<const char*>(a.k);
  p.v = static_cast<const char*>(a.v);
  p.sk = static_cast<const char*>(a.shared_k);
  p.sv = static_cast<const char*>(a.shared_v);
  p.out = static_cast<char*>(a.out);
  p.q_off = a.q_offsets;
  p.k_off = a.k_offsets;
  p.visible = a.visible;
  p.lengths = a.lengths;
  p.pages = a.pages;
  p.slopes = a.slopes;
  p.part = static_cast<float*>(a.workspace);
  p.q_seq = a.q_seq * size;
  p.q_tok = a.q_token * size;
  p.q_head = a.q_head * size;
  p.k_seq = a.k_seq * size;
  p.k_head = a.k_head * size;
  p.v_seq = a.v_seq * size;
  p.v_head = a.v_head * size;
  p.sk_head = a.shared_k_head * size;
  p.sv_head = a.shared_v_head * size;
  p.k_tok = static_cast<uint32_t>(a.k_token * size);
  p.v_tok = static_cast<uint32_t>(a.v_token * size);
  p.sk_tok = static_cast<uint32_t>(a.shared_k_token * size);
  p.sv_tok = static_cast<uint32_t>(a.shared_v_token * size);
  p.seqs = a.seqs;
  p.q_len = a.q_len;
  p.k_len = a.k_len;
  p.hq = a.hq;
  p.hkv = a.hkv;
  p.group = a.hq / a.hkv;
  p.d = a.d;
  p.shared = a.shared;
  p.causal = a.causal != 0;
  p.page = a.page;
  p.max_pages = a.max_pages;
  p.num_pages = a.num_pages;
  p.scale = a.scale > 0.f ? a.scale : (a.scale < 0.f ? -a.scale : 1.f);
  p.sign = a.scale > 0.f ? 1.f : (a.scale < 0.f ? -1.f : 0.f);
  p.softcap = a.softcap;
  return p;
}

// Tiles of 32 keys that a workgroup of four wavefronts on their own keys gets at least.
constexpr int kLeastKeys = 16;

// Splits of `tiles` key tiles so that `items` workgroups become about `many`, with at least `least` tiles a
// split.
int splits_for(int64_t items, int64_t tiles, int many, int least) {
  if (items <= 0 || tiles <= 0) return 1;
  int64_t s = (many + items - 1) / items;
  if (s > tiles / least) s = tiles / least;
  return s < 1 ? 1 : static_cast<int>(s > 256 ? 256 : s);
}

// Places of a row that the products of 128 rows go over (see rows_workgroup).
int places_of(int d) { return d <= 64 ? (d <= 32 ? 32 : 64) : (d <= 96 ? 96 : 128); }

// What a prompt takes in one shape and number of splits, in us. A CU gets through so many steps (tiles of 64 fp16
// or 32 fp32 keys; 128 keys for the four wavefronts of 32 rows) in a time that two workgroups on it mostly share;
// a split's sums go through the workspace and a second launch. Measured for this, us (causal unless said otherwise,
// query heads on key heads): 3 x 597 tokens, 32 on 8 of 128, no mask: 35 whole, 76 in two splits; 4 x 1611, 6 on 2,
// no mask: 60 and 82; 512, 32 on 8: 12.8 in 32 rows, 18 in 128, 31 in two splits; 2048, 8 on 2: 26 in 32 rows, 48 in
// 128, 37 in four splits; 128 rows on 16128 keys, 32 on 8: 60 in 16 splits, 69 in 8, 70 in 32 rows and 4; 2 x 298 after
// 2531, 2 on 2: 18 in 32 rows and 4 splits, 20 in 128 and 16. fp32: 46 x 35, 20 on 5 of 80: 54 in 32 rows, 14 in 128; 2048,
// 32 on 8 of 128: 397 in 128 rows, 297 in two splits, 394 in 32 rows; 4 x 1611, 6 on 2 of 64, no mask: 131 in 32 rows,
// 181 in 128, 141 in four splits; 128 after 3872, 16 heads of 128: 57 in 32 rows and 4 splits, 72 in 128 and 16;
// 32 x 256, 12 heads of 64, no mask: 60 in 128 rows, 85 in 32; 1000, the same: 37 in 32 rows, 52 in 128 and 4 splits.
struct Step {
  float alone, shared, beside;  // one workgroup on a CU; each of several; the longest of several
};
// places: of a row, that the products go over
Step step_of(bool keys, bool f32, int dp, int places) {
  if (f32) {
    if (keys) return dp == 64 ? Step{2.4f, 2.1f, 2.7f} : Step{5.2f, 5.5f, 5.2f};
    if (dp == 64) return places == 32 ? Step{1.6f, 1.f, 1.6f} : Step{2.4f, 2.08f, 3.2f};
    return places == 96 ? Step{3.5f, 2.9f, 4.7f} : Step{4.8f, 3.8f, 6.2f};
  }
  if (keys) return dp == 64 ? Step{0.7f, 0.6f, 0.7f} : Step{0.9f, 0.8f, 0.9f};
  return dp == 64 ? Step{0.9f, 0.55f, 0.9f} : Step{1.45f, 1.2f, 1.45f};
}
float prompt_time(bool keys, bool f32, int d, int64_t items, int64_t steps, float average, int splits, int cus) {
  const int dp = d <= 64 ? 64 : 128;
  const Step t = step_of(keys, f32, dp, places_of(d));
  const int64_t workgroups = items * splits, each = (steps + splits - 1) / splits, share = (workgroups + cus - 1) / cus;
  const float mean = average / static_cast<float>(splits) > 1.f ? average / static_cast<float>(splits) : 1.f;
  // (a CU's share of workgroups: the largest and the mean one, as CUs with fewer leave memory and power to the rest)
  const float part = share > 1 ? 0.5f * (static_cast<float>(share) + static_cast<float>(workgroups) / static_cast<float>(cus)) : 1.f;
  const float longest = static_cast<float>(each) * (share > 1 ? t.beside : t.alone), all = part * mean * t.shared;
  const int at_once = keys && f32 && dp == 128 ? 1 : 2;  // on a CU; further ones start after them
  float us = (keys ? 6.5f : 8.f) + (longest > all ? longest : all);
  if (share > at_once) us += (at_once == 1 ? 5.f : 2.f) * static_cast<float>(share - at_once);
  // (what is written and read again, at 5 TB/s)
  if (splits > 1) us += 4.f + static_cast<float>(workgroups) * static_cast<float>(slot_floats(keys ? kKeyTile : kRowTile, dp)) * 1.6e-6f;
  return us;
}

bool fits_grid(int64_t workgroups) { return workgroups <= (1LL << 24) - 1; }  // 2^32 threads a launch

struct PromptPlan {
  bool keys;
  int rt, tiles, splits;  // splits 0: no shape whose launches are small enough
  size_t bytes;
};
PromptPlan plan_prompt(const g16_attention_args& a) {
  PromptPlan r = {};
  const int group = a.hq / a.hkv, dp = a.d <= 64 ? 64 : 128, cus = cus_of(a);
  const int64_t rows = a.q_offsets == nullptr ? static_cast<int64_t>(a.q_len) * group : static_cast<int64_t>(a.q_len) * group / a.seqs;
  // keys of an average sequence (packed lengths are known on the device only), and what its rows see on average
  const int64_t own = a.q_offsets == nullptr ? a.k_len : a.k_len / a.seqs, keys = a.shared + own;
  const int64_t tokens = a.q_offsets == nullptr ? a.q_len : a.q_len / a.seqs;
  const float seen = static_cast<float>(keys) - (a.causal ? 0.5f * static_cast<float>(tokens < own ? tokens : own) : 0.f);
  float best = 0.f;
  for (int m = 0; m < 2; ++m) {
    const bool by_keys = m == 1;
    const int rt = by_keys ? kKeyTile : kRowTile, step = by_keys ? 128 : (a.is_f32 ? 32 : 64);
    const int64_t items = (rows + rt - 1) / rt * a.seqs * a.hkv, steps = (keys + step - 1) / step;
    // row tiles; packed: at most
    const int64_t tiles = a.q_offsets == nullptr ? (rows + rt - 1) / rt * a.seqs : static_cast<int64_t>(a.q_len) * group / rt + a.seqs;
    for (int s = 1; s <= 256; s = s < 4 ? s + 1 : (s & (s - 1) ? s / 3 * 4 : s / 2 * 3)) {  // 1 2 3 4 6 8 12 16 ..
      if (s > 1 && steps / s < (by_keys ? 1 : 2)) break;
      if (!fits_grid(tiles * s * a.hkv) || (s > 1 && !fits_grid(tiles * a.hkv * (rt / kJoinRows)))) break;
      const float us = prompt_time(by_keys, a.is_f32 != 0, a.d, items, steps, seen / static_cast<float>(step), s, cus);
      if (r.splits > 0 && us >= best) continue;
      best = us;
      r.keys = by_keys;
      r.rt = rt;
      r.tiles = static_cast<int>(tiles);
      r.splits = s;
    }
  }
  if (r.splits > 1) r.bytes = static_cast<size_t>(r.tiles) * r.splits * a.hkv * slot_floats(r.rt, dp) * sizeof(float);
  return r;
}

struct DecodePlan {
  bool skeys, join;
  int stiles, ssplits, otiles, oitems, least;
  int64_t own;  // workgroups a key head for the own keys
  size_t bytes;
};
DecodePlan plan_decode(const g16_attention_args& a) {
  DecodePlan r = {};
  const int group = a.hq / a.hkv, dp = a.d <= 64 ? 64 : 128, cus = cus_of(a);
  const int64_t rows = static_cast<int64_t>(a.seqs) * group;
  r.skeys = rows <= 2 * kKeyTile;
  const int srt = r.skeys ? kKeyTile : kRowTile, sbn = r.skeys || a.is_f32 ? 32 : 64;
  r.stiles = a.shared > 0 ? static_cast<int>((rows + srt - 1) / srt) : 0;
  // (two workgroups a CU; 128 rows of more than 64 values: one, as a second one adds no speed and the requests' own
  // keys take its place: 64 requests, 32768 shared keys, 8 heads of 128: 75 us, with two 83; of 64: 42 and 39.)
  // 32 rows of more than 64 fp32 values: the LDS holds one workgroup a CU, all of which should start at once, and a
  // tile takes five times as long as in fp16, so shorter splits pay (4 requests of up to 1000, 2000 shared, 8 heads of
  // 128: 27.6 us in 10 splits, 42.7 in 3; 11 of up to 22, 11081, 2 of 72: 24.8 in 48, 36 in 21).
  r.otiles = (group + kKeyTile - 1) / kKeyTile;
  const bool single = r.skeys && a.is_f32 && dp == 128;
  const int64_t others = a.seqs * static_cast<int64_t>(r.otiles) * a.hkv;
  const int many = single ? static_cast<int>(others < cus / 2 ? cus - others : cus / 2) : (r.skeys || dp == 64 ? 2 * cus : cus);
  r.ssplits = splits_for(static_cast<int64_t>(r.stiles) * a.hkv, (a.shared + sbn - 1) / sbn, many, single ? 6 : (r.skeys ? kLeastKeys : 4));
  const int64_t items = (2 * cus + static_cast<int64_t>(r.otiles) * a.hkv - 1) / (static_cast<int64_t>(r.otiles) * a.hkv);
  // (at most as many parts as there are requests: one each, and no need to look for it)
  const bool split = (a.k_len + 31) / 32 > kLeastKeys && items > 1;
  r.oitems = static_cast<int>(items);
  // (8 x 8 heads' parts of 16 requests up to 1500 keys: 24.8 us with 16 tiles at least, 22.4 with 8)
  r.least = split ? kLeastKeys / 2 : 0;
  r.own = (split ? items + a.seqs : a.seqs) * r.otiles;
  r.join = r.stiles > 0 || split;
  if (r.join)
    r.bytes = (static_cast<size_t>(r.stiles) * r.ssplits * a.hkv * slot_floats(srt, dp) +
               static_cast<size_t>(r.own) * a.hkv * slot_floats(own_rows(group), dp)) * sizeof(float);
  return r;
}

template <typename T, int DP>
int run_prompt(const Params& p, const PromptPlan& plan, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(plan.tiles) * plan.splits * p.hkv);
  constexpr int kLess = DP == 64 ? 32 : 96;
  int rc = plan.keys      ? launch(prompt_kernel<T, DP, DP, true>, grid, dim3(kThreads), stream, p)
           : places_of(p.d) == kLess ? launch(prompt_kernel<T, DP, kLess, false>, grid, dim3(kThreads), stream, p)
                          : launch(prompt_kernel<T, DP, DP, false>, grid, dim3(kThreads), stream, p);
  if (rc == 0 && plan.splits > 1)
    rc = launch(prompt_join_kernel<T, DP>, dim3(static_cast<unsigned>(plan.tiles) * p.hkv * (plan.rt / kJoinRows)), dim3(kThreads), stream, p,
                plan.rt);
  return rc;
}
template <typename T, int DP>
int run_decode(const Params& p, const DecodePlan& plan, hipStream_t stream) {
  const dim3 grid((static_cast<unsigned>(p.stiles) * p.ssplits + static_cast<unsigned>(plan.own)) * p.hkv);
  int rc = plan.skeys ? launch(decode_kernel<T, DP, true>, grid, dim3(kThreads), stream, p)
                      : launch(decode_kernel<T, DP, false>, grid, dim3(kThreads), stream, p);
  if (rc == 0 && plan.join)
    rc = launch(decode_join_kernel<T, DP>, dim3(static_cast<unsigned>((static_cast<int64_t>(p.seqs) * p.hq + 3) / 4)), dim3(kThreads), stream, p,
                plan.skeys ? kKeyTile : kRowTile);
  return rc;
}

int check8(const g16_attention8_args& e) {
  const int st = check(e.a, true, true);
  if (e.code != G16_CODE_INT8 && e.code != G16_CODE_E4M3) return G16_E_DTYPE;
  if (st != G16_OK || e.a.seqs == 0 || e.a.hq == 0) return st;
  return e.a.k_len > 0 && (e.k_scale == nullptr || e.v_scale == nullptr) ? G16_E_NULL : G16_OK;
}

// The own keys' part of the plan for a cache in 8 bits (see attention8.hip), and what the workspace has to hold.
struct Plan8 {
  DecodePlan shared;
  int heads, shares;
  bool split;
  size_t table;         // floats of the requests' table, before the slots
  size_t first, bytes;  // floats before the own keys' slots; bytes in all
};
Plan8 plan_decode8(const g16_attention_args& a) {
  Plan8 r = {};
  r.shared = plan_decode(a);
  const int group = a.hq / a.hkv, dp = a.d <= 64 ? 64 : 128, srt = r.shared.skeys ? kKeyTile : kRowTile;
  const int64_t heads = static_cast<int64_t>(r.shared.otiles) * a.hkv;
  r.split = a.k_len > kWhole8 * kTile8;
  r.shares = a.seqs;
  r.heads = 1;
  if (r.split) {
    // as many as run at once, the same number for every XCD
    auto shares = [&](int together) {
      const int64_t each = static_cast<int64_t>(cus_of(a)) / kXcds * waves_of8(a.is_f32 != 0, dp, rows_of8(group)) * together / heads;
      return static_cast<int>(each < 1 ? kXcds : each * kXcds);
    };
    // Where a token's heads lie next to each other in memory, a workgroup takes four of them together (see own8_workgroup), unless
    // there are so few requests that their joins would take longer (one request of 8192 keys, 32 heads on 8, d 128, 256 parts of a row:
    // 19.9 us, 18.5 by single heads; 16 heads on 16, 128 parts: 18.8 and 19.6, of 65536 69.2 and 76.7; two requests of 8192, 64 heads on 8,
    // 128 parts: 23.9 and 21.8; 64 of up to 700, 32 heads on 8: 24.7 and 30.8; all in graphs).
    if (a.hkv % kHeads8 == 0 && rows_of8(group) <= kRowsOfHeads8 && a.d == dp && a.k_token > a.k_head && shares(kHeads8) <= 128LL * a.seqs) r.heads = kHeads8;
    r.shares = shares(r.heads);
  }
  const bool join = r.shared.stiles > 0 || r.split;
  r.table = join ? (static_cast<size_t>(a.seqs) * sizeof(Slots) + 15) / 16 * 4 : 0;
  r.first = r.table + static_cast<size_t>(r.shared.stiles) * r.shared.ssplits * a.hkv * slot_floats(srt, dp);
  if (join)
    r.bytes = (r.first + (static_cast<size_t>(r.shares) + (r.split ? a.seqs : 0)) * heads * slot_floats(own_rows(group), dp)) * sizeof(float);
  return r;
}

// Whether shared and own keys go into one launch: few enough kernels, and with two workgroups on a CU as many as either would
// have by itself, or nearly: for heads of 64 the own keys' shares are counted for three (counting two: 16.4 us for 16.3, 16 requests
// of up to 1500 after 2048, 12 heads of 64).
bool both8(const g16_attention_args& a, const Plan8& plan) {
  return plan.shared.stiles > 0 && plan.shared.skeys && !a.is_f32 && (a.d == 64 || a.d == 128) && a.hq / a.hkv <= 8;
}
template <int DP, int CODE, int HEADS>
int run_both8(const Params& p, const Params8& e, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(p.stiles) * p.ssplits * p.hkv + workgroups_of8(p, e));
  return p.group == 1   ? launch(decode_both8_kernel<DP, CODE, 1, HEADS>, grid, dim3(kThreads), stream, p, e)
         : p.group <= 4 ? launch(decode_both8_kernel<DP, CODE, 4, HEADS>, grid, dim3(kThreads), stream, p, e)
                        : launch(decode_both8_kernel<DP, CODE, 8, HEADS>, grid, dim3(kThreads), stream, p, e);
}
template <int DP, int CODE>
int run_both8(const Params& p, const Params8& e, hipStream_t stream) {
  return e.heads == 1 ? run_both8<DP, CODE, 1>(p, e, stream) : run_both8<DP, CODE, kHeads8>(p, e, stream);
}

template <typename T, int DP>
int run_shared8(const Params& p, bool skeys, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(p.stiles) * p.ssplits * p.hkv);
  return skeys ? launch(decode_kernel<T, DP, true>, grid, dim3(kThreads), stream, p) : launch(decode_kernel<T, DP, false>, grid, dim3(kThreads), stream, p);
}

}  // namespace
}  // namespace g16

using namespace g16;

extern "C" size_t g16_attention_workspace_bytes(const g16_attention_args* args) {
  if (args == nullptr || check(*args, false) != G16_OK || args->seqs == 0 || args->hq == 0 || args->q_len == 0) return 0;
  return plan_prompt(*args).bytes;
}

extern "C" int g16_attention_plan(const g16_attention_args* args, int* row_tile, int* splits) {
  if (args == nullptr || row_tile == nullptr || splits == nullptr) return G16_E_NULL;
  *row_tile = *splits = 0;
  const int st = check(*args, false);
  if (st != G16_OK || args->seqs == 0 || args->hq == 0 || args->q_len == 0) return st;
  const PromptPlan plan = plan_prompt(*args);
  if (plan.splits == 0) return G16_E_SHAPE;
  *row_tile = plan.rt;
  *splits = plan.splits;
  return G16_OK;
}

extern "C" int g16_attention(const g16_attention_args* args, void* stream) {
  if (args == nullptr) return G16_E_NULL;
  const g16_attention_args& a = *args;
  const int st = check(a, false);
  if (st != G16_OK || a.seqs == 0 || a.hq == 0 || a.q_len == 0) return st;
  const PromptPlan plan = plan_prompt(a);
  if (plan.splits == 0) return G16_E_SHAPE;
  if (plan.bytes > 0 && (a.workspace == nullptr || static_cast<size_t>(a.workspace_bytes) < plan.bytes)) return G16_E_WORKSPACE;
  if (!aligned16(a.workspace)) return G16_E_ALIGN;
  Params p = params(a);
  p.tiles = plan.tiles;
  p.splits = plan.splits;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a.is_f32) return a.d <= 64 ? run_prompt<float, 64>(p, plan, s) : run_prompt<float, 128>(p, plan, s);
  return a.d <= 64 ? run_prompt<_Float16, 64>(p, plan, s) : run_prompt<_Float16, 128>(p, plan, s);
}

extern "C" size_t g16_attention_decode_workspace_bytes(const g16_attention_args* args) {
  if (args == nullptr || check(*args, true) != G16_OK || args->seqs == 0 || args->hq == 0) return 0;
  return plan_decode(*args).bytes;
}

extern "C" int g16_attention_decode(const g16_attention_args* args, void* stream) {
  if (args == nullptr) return G16_E_NULL;
  const g16_attention_args& a = *args;
  const int st = check(a, true);
  if (st != G16_OK || a.seqs == 0 || a.hq == 0) return st;
  const DecodePlan plan = plan_decode(a);
  if (plan.bytes > 0 && (a.workspace == nullptr || static_cast<size_t>(a.workspace_bytes) < plan.bytes)) return G16_E_WORKSPACE;
  if (!aligned16(a.workspace)) return G16_E_ALIGN;
  if (!fits_grid((static_cast<int64_t>(plan.stiles) * plan.ssplits + plan.own) * a.hkv) ||
      !fits_grid((static_cast<int64_t>(a.seqs) * a.hq + 3) / 4))
    return G16_E_SHAPE;
  Params p = params(a);
  p.causal = 0;
  p.stiles = plan.stiles;
  p.ssplits = plan.ssplits;
  p.otiles = plan.otiles;
  p.oitems = plan.oitems;
  p.least = plan.least;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a.is_f32) return a.d <= 64 ? run_decode<float, 64>(p, plan, s) : run_decode<float, 128>(p, plan, s);
  return a.d <= 64 ? run_decode<_Float16, 64>(p, plan, s) : run_decode<_Float16, 128>(p, plan, s);
}

extern "C" size_t g16_attention_decode8_workspace_bytes(const g16_attention8_args* args) {
  if (args == nullptr || check8(*args) != G16_OK || args->a.seqs == 0 || args->a.hq == 0) return 0;
  return plan_decode8(args->a).bytes;
}

extern "C" int g16_attention_decode8(const g16_attention8_args* args, void* stream) {
  if (args == nullptr) return G16_E_NULL;
  const g16_attention8_args& e = *args;
  const g16_attention_args& a = e.a;
  const int st = check8(e);
  if (st != G16_OK || a.seqs == 0 || a.hq == 0) return st;
  if (static_cast<int64_t>(a.seqs) * (a.k_len / kTile8 + 1) > (1LL << 31) - 1) return G16_E_SHAPE;  // (tiles are counted in 32 bits)
  const Plan8 plan = plan_decode8(a);
  if (plan.bytes > 0 && (a.workspace == nullptr || static_cast<size_t>(a.workspace_bytes) < plan.bytes)) return G16_E_WORKSPACE;
  if (!aligned16(a.workspace)) return G16_E_ALIGN;
  if (!fits_grid((static_cast<int64_t>(plan.shared.stiles) * plan.shared.ssplits + (static_cast<int64_t>(plan.shares) + kXcds) * plan.shared.otiles) * a.hkv) || !fits_grid((static_cast<int64_t>(a.seqs) * a.hq + 3) / 4))
    return G16_E_SHAPE;
  Params p = params(a);
  p.causal = 0;
  p.stiles = plan.shared.stiles;
  p.ssplits = plan.shared.ssplits;
  p.otiles = plan.shared.otiles;
  p.part += plan.table;
  p.k_seq = a.k_seq;
  p.k_head = a.k_head;
  p.v_seq = a.v_seq;
  p.v_head = a.v_head;
  const Params8 own = {e.k_scale, e.v_scale, e.ks_seq, e.ks_head, e.ks_token, e.vs_seq, e.vs_head, e.vs_token, a.k_token, a.v_token,
                       divide_by(a.page > 0 ? static_cast<uint32_t>(a.page) : 1u), plan.heads, plan.shares, plan.split, plan.shared.skeys ? kKeyTile : kRowTile, !both8(a, plan), plan.first - plan.table,
                       plan.bytes > 0 ? static_cast<Slots*>(a.workspace) : nullptr};
  hipStream_t s = static_cast<hipStream_t>(stream);
  int rc = 0;
  if (!own.apart) {
    if (e.code == G16_CODE_INT8) rc = a.d == 64 ? run_both8<64, G16_CODE_INT8>(p, own, s) : run_both8<128, G16_CODE_INT8>(p, own, s);
    else rc = a.d == 64 ? run_both8<64, G16_CODE_E4M3>(p, own, s) : run_both8<128, G16_CODE_E4M3>(p, own, s);
  } else if (p.stiles > 0) {
    if (a.is_f32) rc = a.d <= 64 ? run_shared8<float, 64>(p, plan.shared.skeys, s) : run_shared8<float, 128>(p, plan.shared.skeys, s);
    else rc = a.d <= 64 ? run_shared8<_Float16, 64>(p, plan.shared.skeys, s) : run_shared8<_Float16, 128>(p, plan.shared.skeys, s);
  }
  return rc == 0 ? run_own8(p, own, e.code, a.is_f32 != 0, s) : rc;
}
