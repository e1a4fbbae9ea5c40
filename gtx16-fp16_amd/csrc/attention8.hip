// Single tokens over a cache of 8 bits: the launches for the requests' own keys (attention8_own.hpp) and the joins of their sums
// and the shared keys'.
#include "attention8_own.hpp"

namespace g16 {
namespace {

// A row's slots: of the shared keys, then of its request's pieces in shares one after another. W wavefronts have a row's slots
// among them: four where there are few rows, whose time is that of the longest (a call with 64 slots for each of 32 rows of 128
// values: 62.8 us with one, so 59.9; with 128 rows 38.3 and 33.3; but 512 rows of few slots 22.3 and 23.3).
template <typename T, int DP, int W>
__global__ __launch_bounds__(kThreads) void decode8_join_kernel(Params p, Params8 e) {
  __shared__ __attribute__((aligned(16))) float sums[W == 1 ? 1 : 4][DP + 4];
  const int wave = uniform(static_cast<int>(threadIdx.x >> 6));
  const int row = W == 1 ? static_cast<int>(blockIdx.x) * 4 + wave : static_cast<int>(blockIdx.x);
  if (row >= p.seqs * p.hq) return;
  const int b = row / p.hq, head = row % p.hq, kv = head / p.group, g = head % p.group;
  const int ns = p.stiles > 0 ? p.ssplits : 0, orows = own_rows(p.group), sr = b * p.group + g;
  const Slots own = e.table[b];
  const int parts = ns + own.count;
  if (parts == 1) return;
  auto slot_of = [&](int i, const float*& o, const float*& m, int& rows) {
    const float* slot;
    int r;
    if (i < ns) {
      slot = p.part + (static_cast<size_t>((sr / e.srt) * p.ssplits + i) * p.hkv + kv) * slot_floats(e.srt, DP);
      r = sr % e.srt;
      rows = e.srt;
    } else {
      const size_t at = (static_cast<size_t>(own.first) + (i - ns)) * p.otiles + g / kKeyTile;
      slot = p.part + e.first + (at * p.hkv + kv) * slot_floats(orows, DP);
      r = g % kKeyTile;
      rows = orows;
    }
    o = slot + static_cast<size_t>(r) * DP;
    m = slot + static_cast<size_t>(rows) * DP + r;
  };
  char* out = p.out + static_cast<int64_t>(row) * p.d * static_cast<int>(sizeof(T));
  if constexpr (W == 1) {
    join_row<T, DP>(out, p.d, parts, slot_of);
  } else {
    const int from = share_begin(parts, wave, 4), mine = share_begin(parts, wave + 1, 4) - from;
    float top = -__builtin_huge_valf(), l = 0.f;
    float4v o = {};
    if (mine > 0) join_sums<DP>(mine, [&](int i, const float*& s, const float*& m, int& rows) { slot_of(from + i, s, m, rows); }, top, l, o);
    const int lane = threadIdx.x & 63, d0 = lane % (DP / 4) * 4;
    if (lane < DP / 4) *reinterpret_cast<float4v*>(&sums[wave][d0]) = o;
    if (lane == 0) {
      sums[wave][DP] = top;
      sums[wave][DP + 1] = l;
    }
    __syncthreads();
    if (wave != 0 || lane >= DP / 4 || d0 >= p.d) return;
    top = fmaxf(fmaxf(sums[0][DP], sums[1][DP]), fmaxf(sums[2][DP], sums[3][DP]));
    l = 0.f;
    o = float4v{};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float f = sums[i][DP] == top ? 1.f : __builtin_amdgcn_exp2f(sums[i][DP] - top);
      l = fmaf(f, sums[i][DP + 1], l);
      o += f * *reinterpret_cast<const float4v*>(&sums[i][d0]);
    }
    const float inv = inverse(l), r[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
    store_out<T, 4>(out, d0, r);
  }
}

template <typename T, int DP, int CODE, int RQ, bool FULL, int HEADS>
__global__ __launch_bounds__(kThreads, waves_of8(sizeof(T) == 4, DP, RQ)) void decode8_kernel(Params p, Params8 e) {
  __shared__ Lds8<T, DP, RQ> lds;
  own8_workgroup<T, DP, CODE, RQ, FULL, HEADS>(p, e, static_cast<int>(blockIdx.x), lds);
}

template <typename T, int DP, int CODE, int RQ>
int run(const Params& p, const Params8& e, dim3 grid, hipStream_t stream) {
  if constexpr (RQ <= kRowsOfHeads8) {
    if (e.heads == kHeads8) return launch(decode8_kernel<T, DP, CODE, RQ, true, kHeads8>, grid, dim3(kThreads), stream, p, e);
  }
  return p.d == DP ? launch(decode8_kernel<T, DP, CODE, RQ, true, 1>, grid, dim3(kThreads), stream, p, e)
                   : launch(decode8_kernel<T, DP, CODE, RQ, false, 1>, grid, dim3(kThreads), stream, p, e);
}
template <typename T, int DP>
int join(const Params& p, const Params8& e, hipStream_t stream) {
  if (p.stiles == 0 && !e.split) return 0;
  const unsigned rows = static_cast<unsigned>(p.seqs) * p.hq;
  return rows <= 512 ? launch(decode8_join_kernel<T, DP, 4>, dim3(rows), dim3(kThreads), stream, p, e)
                     : launch(decode8_join_kernel<T, DP, 1>, dim3((rows + 3) / 4), dim3(kThreads), stream, p, e);
}
template <typename T, int DP, int CODE>
int run(const Params& p, const Params8& e, hipStream_t stream) {
  const dim3 grid(workgroups_of8(p, e));
  int rc = 0;
  if (!e.apart) return join<T, DP>(p, e, stream);
  switch (rows_of8(p.group)) {
    case 1: rc = run<T, DP, CODE, 1>(p, e, grid, stream); break;
    case 4: rc = run<T, DP, CODE, 4>(p, e, grid, stream); break;
    case 8: rc = run<T, DP, CODE, 8>(p, e, grid, stream); break;
    case 16: rc = run<T, DP, CODE, 16>(p, e, grid, stream); break;
    default: rc = run<T, DP, CODE, 32>(p, e, grid, stream);
  }
  return rc == 0 ? join<T, DP>(p, e, stream) : rc;
}
template <typename T>
int run(const Params& p, const Params8& e, int code, hipStream_t stream) {
  if (code == G16_CODE_INT8) return p.d <= 64 ? run<T, 64, G16_CODE_INT8>(p, e, stream) : run<T, 128, G16_CODE_INT8>(p, e, stream);
  return p.d <= 64 ? run<T, 64, G16_CODE_E4M3>(p, e, stream) : run<T, 128, G16_CODE_E4M3>(p, e, stream);
}

}  // namespace

int run_own8(const Params& p, const Params8& e, int code, bool f32, hipStream_t stream) {
  return f32 ? run<float>(p, e, code, stream) : run<_Float16>(p, e, code, stream);
}

}  // namespace g16
