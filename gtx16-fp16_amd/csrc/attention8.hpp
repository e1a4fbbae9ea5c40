// Single tokens over a cache of 8 bits (g16_attention_decode8); part of attention.hip, whose rows, scores, parts, slots and joins it
// shares. The shared prefix is not in 8 bits and decode_kernel's own.
//
// A wavefront has 16 or 32 query rows of one key head and tiles of 32 keys of its own, straight from memory into registers:
//   * S^T = K Q^T in 16x16x32 blocks: lane l holds keys 4 (l / 16) + {0..3} of a block and query row l % 16. Lane l's key of the
//     first operand is l % 16, and its values come in 16-byte loads, 64 bytes of a key an instruction: a step's values are
//     bytes 8 of that piece, in another order than in memory, the queries' too.
//   * O^T += V^T P^T with 32 keys a step: the weights leave the first product in the order in which the second one wants
//     them, if its step takes keys 4 (l / 16) + {0..3} and 16 + 4 (l / 16) + {0..3} from lane l. Lane l loads DP / 16 values of
//     each of these eight keys, from value (l % 16) DP / 16 on: a key's row is one run of an instruction. Byte b of the
//     eight loads makes the operand of block b, so the transposition costs nothing but the choice of bytes, and block
//     b's row m is value m DP / 16 + b.
//   * Codes are exact in fp16 and bf16. K is multiplied as fp16 where the queries are, else as bf16 with the queries in three
//     parts. A key's scale joins its score; a value's joins its weight, whose range then is fp32's, so weights are multiplied as
//     bf16 parts: two for fp16 (to 2^-17; results are 2.1e-4 from the exact ones, all of it their own rounding), three for fp32.
//     So that the last of three is no subnormal, which the products take for 0, fp32's sums are kept in a unit: the power of
//     two of the largest scale so far, within 2^40.
//   * The places of a tile's rows are found one key a lane, a tile ahead of its loads and two ahead of its products, and
//     passed on through 512 bytes of LDS a wavefront, as are the scales.
// A key behind its request's end, or on a page outside the cache, is read from a row of zeros; the former get no weight.

struct Params8 {
  const float *ks, *vs;
  int64_t ks_seq, ks_head, ks_tok, vs_seq, vs_head, vs_tok;  // elements
  int64_t k_tok, v_tok;                                      // bytes
  size_t first;                                              // floats of the shared keys' slots, before these parts'
};

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
    return mma16(halves<CODE>(codes), v, c);
  }
};
template <>
struct Query8<float> {
  Split8 v;
  __device__ void set(float8v x) { v = operand_of_any(x); }
  // (the small products first, as in products_as)
  template <int CODE>
  __device__ float4v times(u32x2 codes, float4v c) const {
    const bhalf8 k = bfloats<CODE>(codes);
    return mma16(k, v.hi, mma16(k, v.mid, mma16(k, v.lo, c)));
  }
};

// A tile of 32 keys as it is loaded.
template <int DP>
struct Raw8 {
  static constexpr int KW = DP / 16, VW = DP / 64;  // dwords of a lane's piece of a key, of a value
  uint32_t k[2][KW], v[8][VW];
  float scale;  // of key lane % 32: its key's, or, in the upper lanes, its value's
};

template <typename T, int DP, int CODE, int NR, bool FULL>
__global__ __launch_bounds__(kThreads, 2) void decode8_kernel(Params p, Params8 e) {
  constexpr int VB = DP / 16;  // values of a lane, blocks of the second product
  constexpr int R = 16 * NR;
  __shared__ __attribute__((aligned(16))) float so[4 * R * DP];
  __shared__ __attribute__((aligned(16))) uint64_t places[4][64];
  __shared__ __attribute__((aligned(16))) float scales[4][64];
  __shared__ float joint[2][4][R];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 15, g = lane >> 4;
  int lin = blockIdx.x;
  const int own = lin;
  const int kv = lin % p.hkv;
  lin /= p.hkv;
  const int rt = lin % p.otiles;
  Part part;
  if (!find_part(p, lin / p.otiles, true, part)) return;
  const int b = part.seq, len = part.len, orows = own_rows(p.group);
  const Scoring sc = scoring(p);
  const int n = ceil_div(len, 32);
  const int tbeg = share_begin(n, part.split, part.splits), tend = share_begin(n, part.split + 1, part.splits);

  // ---- this lane's key of a tile ----
  const bool upper = lane >= 32;
  const int32_t* table = p.pages == nullptr ? nullptr : p.pages + static_cast<size_t>(b) * p.max_pages;
  const char* base = upper ? p.v + kv * p.v_head : p.k + kv * p.k_head;
  const float* sbase = upper ? e.vs + kv * e.vs_head : e.ks + kv * e.ks_head;
  const int64_t seq = upper ? p.v_seq : p.k_seq, tok = upper ? e.v_tok : e.k_tok;
  const int64_t sseq = upper ? e.vs_seq : e.ks_seq, stok = upper ? e.vs_tok : e.ks_tok;
  auto page_of = [&](int t) {  // -1: no such key
    const int j = 32 * t + (lane & 31);
    int pg = -1;
    if (t < tend && j < len) {
      pg = b;
      if (table != nullptr) {
        pg = table[j / p.page];
        if (static_cast<unsigned>(pg) >= static_cast<unsigned>(p.num_pages)) pg = -1;
      }
    }
    return pg;
  };
  Raw8<DP> raw;
  auto load = [&](int t, int pg) {
    const int j = 32 * t + (lane & 31), at = table != nullptr ? j % p.page : j;
    const char* row = pg < 0 ? reinterpret_cast<const char*>(g_zero_row) : base + pg * seq + at * tok;
    places[wave][lane] = reinterpret_cast<uint64_t>(row);
    raw.scale = pg < 0 ? 0.f : sbase[pg * sseq + at * stok];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const char* k = reinterpret_cast<const char*>(places[wave][16 * s + col]);
#pragma unroll
      for (int c = 0; c < DP / 64; ++c) {
        const int at0 = 64 * c + 16 * g;
        if constexpr (FULL) {
          struct alignas(8) Piece {
            uint32_t w[4];
          };
          const Piece x = *reinterpret_cast<const Piece*>(k + at0);
#pragma unroll
          for (int w = 0; w < 4; ++w) raw.k[s][4 * c + w] = x.w[w];
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const bool some = at0 + 8 * h < p.d;
            const u32x2 x = *reinterpret_cast<const u32x2*>(k + (some ? at0 + 8 * h : 0));
            raw.k[s][4 * c + 2 * h] = some ? x[0] : 0;
            raw.k[s][4 * c + 2 * h + 1] = some ? x[1] : 0;
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const char* v = reinterpret_cast<const char*>(places[wave][32 + 16 * (i >> 2) + 4 * g + (i & 3)]);
      const bool some = FULL || col * VB < p.d;
      if constexpr (VB == 8) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(v + (some ? col * 8 : 0));
        raw.v[i][0] = some ? x[0] : 0;
        raw.v[i][1] = some ? x[1] : 0;
      } else {
        const uint32_t x = *reinterpret_cast<const uint32_t*>(v + (some ? col * 4 : 0));
        raw.v[i][0] = some ? x : 0;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };

  // ---- this lane's query rows ----
  Query8<T> q[NR][DP / 32];
  float slope[NR], m[NR], l[NR], unit = 0x1p100f;
  float4v o[NR][VB];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int row = rt * kKeyTile + 16 * r + col;
    const bool some = row < p.group;
    const int head = kv * p.group + (some ? row : 0);
    const char* at = p.q + b * p.q_seq + head * p.q_head;
    slope[r] = p.slopes != nullptr ? p.slopes[head] * kLog2e : 0.f;
    m[r] = -__builtin_huge_valf();
    l[r] = 0.f;
#pragma unroll
    for (int s = 0; s < DP / 32; ++s) {
      using V8 = typename Vec8<T>::V;
      const int d0 = 64 * (s >> 1) + 16 * g + 8 * (s & 1);
      V8 x = {};
      if (some && d0 < p.d) x = *reinterpret_cast<const V8*>(at + d0 * sizeof(T));
      if (p.sign != 1.f) x *= static_cast<T>(p.sign);
      q[r][s].set(x);
    }
#pragma unroll
    for (int i = 0; i < VB; ++i) o[r][i] = float4v{};
  }

  int t = tbeg + wave;
  if (t < tend) load(t, page_of(t));
  int next = page_of(t + 4);
  for (; t < tend; t += 4) {
    const Raw8<DP> now = raw;
    scales[wave][lane] = now.scale;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    float ks[8], vs[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      *reinterpret_cast<float4v*>(ks + 4 * h) = *reinterpret_cast<const float4v*>(&scales[wave][16 * h + 4 * g]);
      *reinterpret_cast<float4v*>(vs + 4 * h) = *reinterpret_cast<const float4v*>(&scales[wave][32 + 16 * h + 4 * g]);
    }
    if (t + 4 < tend) load(t + 4, next);
    next = page_of(t + 8);
    if constexpr (sizeof(T) == 4) {
      float most = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(vs[i]));
      if (__any(most * unit > 0x1p40f)) {
        most = fmaxf(most, __shfl_xor(most, 16));
        most = fmaxf(most, __shfl_xor(most, 32));
        const float was = unit;
        unit = __uint_as_float((254u << 23) - (min(__float_as_uint(most), 0x7e800000u) & 0x7f800000u));
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int i = 0; i < VB; ++i) o[r][i] *= unit / was;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) vs[i] *= unit;
    }
    const int left = len - 32 * t;
    float w[NR][8];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        float4v x = {};
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) x = q[r][c].template times<CODE>(u32x2{now.k[s][2 * c], now.k[s][2 * c + 1]}, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[r][4 * s + i] = x[i] * ks[4 * s + i];
      }
      float top = -__builtin_huge_valf();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = 16 * (i >> 2) + 4 * g + (i & 3);
        float x = w[r][i] * sc.c;
        if (sc.capped) {
          if (sizeof(T) == 2 && !sc.fine) x = fmaf(-2.f * sc.cap, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(w[r][i] * sc.inv2)), sc.cap);
          else x = sc.cap * tanh_of(w[r][i] * sc.inv);
        }
        if (sc.biased) x = fmaf(-slope[r], static_cast<float>(left - 1 - j), x);
        w[r][i] = j < left ? x : -__builtin_huge_valf();
        top = fmaxf(top, w[r][i]);
      }
      if (__any(top > m[r] + kLag)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float up = fmaxf(m[r], top);
        const float f = up == m[r] ? 1.f : __builtin_amdgcn_exp2f(m[r] - up);
        m[r] = up;
        l[r] *= f;
#pragma unroll
        for (int i = 0; i < VB; ++i) o[r][i] *= f;
      }
      const float ref = (m[r] == -__builtin_huge_valf() ? 0.f : m[r]) - kShift<T>;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = __builtin_amdgcn_exp2f(w[r][i] - ref) * kScale<T>;
        l[r] += x;
        w[r][i] = x * vs[i];
      }
    }
    bhalf8 part0[NR], part1[NR], part2[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      float8v x;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = w[r][i];
      part0[r] = take_part(x);
      if constexpr (sizeof(T) == 4) {
        part1[r] = take_part(x);
        part2[r] = __builtin_convertvector(x, bhalf8);
      } else {
        part1[r] = __builtin_convertvector(x, bhalf8);
      }
    }
#pragma unroll
    for (int i = 0; i < VB; ++i) {
      uint32_t v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = now.v[k][i >> 2];
      const bhalf8 a = bfloats_of_byte<CODE>(v, i & 3);
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        if constexpr (sizeof(T) == 4) o[r][i] = mma16(a, part2[r], o[r][i]);
        o[r][i] = mma16(a, part1[r], o[r][i]);
        o[r][i] = mma16(a, part0[r], o[r][i]);
      }
    }
  }

  // ---- join the four wavefronts: sums [wave][row][value] in LDS, then eight values a thread ----
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < VB; ++i) o[r][i] *= 1.f / unit;
    }
    l[r] += __shfl_xor(l[r], 16);
    l[r] += __shfl_xor(l[r], 32);
    if (g == 0) {
      joint[0][wave][16 * r + col] = m[r];
      joint[1][wave][16 * r + col] = l[r];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)  // row 4 g + k of every block: values (4 g + k) VB + {0 .. VB - 1}
#pragma unroll
      for (int i = 0; i < VB; i += 4)
        *reinterpret_cast<float4v*>(&so[(wave * R + 16 * r + col) * DP + (4 * g + k) * VB + i]) =
            float4v{o[r][i][k], o[r][i + 1][k], o[r][i + 2][k], o[r][i + 3][k]};
  }
  __syncthreads();
  Slot slot = {nullptr, orows};
  if (p.stiles > 0 || part.splits > 1) slot.at = p.part + e.first + static_cast<size_t>(own) * slot_floats(orows, DP);
  for (int item = tid; item < R * (DP / 8); item += kThreads) {
    const int r = item / (DP / 8), d0 = item % (DP / 8) * 8, row = rt * kKeyTile + r;
    if (row >= p.group) break;
    float top = -__builtin_huge_valf(), f[4], total = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, joint[0][i][r]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float mi = joint[0][i][r];
      f[i] = mi == top ? 1.f : __builtin_amdgcn_exp2f(mi - top);
      total = fmaf(f[i], joint[1][i][r], total);
    }
    const float inv = slot.at != nullptr ? 1.f : inverse(total);
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float x = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) x = fmaf(f[i], so[(i * R + r) * DP + d0 + k], x);
      v[k] = x * inv;
    }
    if (slot.at != nullptr) {
      float* to = slot.at + static_cast<size_t>(r) * DP + d0;
      *reinterpret_cast<float4v*>(to) = float4v{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<float4v*>(to + 4) = float4v{v[4], v[5], v[6], v[7]};
      if (d0 == 0) {
        slot_m<DP>(slot)[r] = top;
        slot_m<DP>(slot)[orows + r] = total;
      }
    } else if (d0 < p.d) {
      store_out<T, 8>(p.out + (static_cast<int64_t>(b) * p.hq + kv * p.group + row) * p.d * static_cast<int>(sizeof(T)), d0, v);
    }
  }
}
