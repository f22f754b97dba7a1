// Appends keys and values to a paged cache, the keys rotated on the way.
//
// New token j of sequence b goes to position lengths[b] + j: row position % page of
// page pages[b][position / page].  K is rotated by the token's table row and rounded
// once to the cache's type; V is copied.  A thread takes 8 channels of one token and
// kAppendHeads key heads, which share one read of the table row.  Bound by memory:
// each new row is read once and written once.  Measured: 8200 tokens, 8 heads, D 128, bf16
// 13.8 us (5.2 TB/s; a large copy reaches 4.9); one token, 12 heads 5.8 us, the launch.
#include "seq.h"

namespace farope {

constexpr int kAppendHeads = 4;

template <typename S, int D>
__global__ void __launch_bounds__(256) cache_append_kernel(const AppendParams p, int n_grp) {
  constexpr int CPR = D / 8, ROWS = 256 / CPR;
  const int blk = block_id() / n_grp, h0 = (block_id() - blk * n_grp) * kAppendHeads;
  const int tid = thread_id(), lane = tid & 63;
  const int t0 = blk * ROWS, t = t0 + tid / CPR, c = 8 * (tid % CPR);
  int b = t, j = 0;
  if (p.cu) {
    const int tc = t < p.T ? t : p.T - 1;
    b = find_seq(p.cu, p.B, p.T, t0, tc, lane);
    j = tc - cu_at(p.cu, b, p.T);
  }
  if (t >= p.T || b >= p.B) return;   // (tokens behind the last sequence are no sequence's)
  const int before = p.c.lengths[b];
  const int64_t pos = (int64_t)before + j, place = pos / p.c.page;
  if (before < 0 || place >= p.c.max_pages) return;
  const int page = p.c.pages[b * p.c.spages + place];
  if (page < 0 || page >= p.c.n_pages) return;   // (not a page of the cache: the token is not stored)
  const int64_t in = pos - place * p.c.page;
  const int64_t index = pos - p.has_cls;
  const int row = table_row(p.positions ? p.positions[t] : (int)(index < INT32_MAX ? index : INT32_MAX), p.n_pos);

  float x[kAppendHeads][8];
  Raw8<S> v[kAppendHeads];
#pragma unroll
  for (int i = 0; i < kAppendHeads; ++i) {
    if (h0 + i >= p.Hkv) break;
    load8<S>(static_cast<const S*>(p.k) + t * p.sk[0] + (h0 + i) * p.sk[1] + c * p.sk[2], p.sk[2], p.vec_k, x[i]);
    v[i] = load_raw8<S>(static_cast<const S*>(p.v) + t * p.sv[0] + (h0 + i) * p.sv[1] + c * p.sv[2], p.sv[2], p.vec_v);
  }
  float cs[8];
  table_load4(p.cosp, p.sinp, row, D / 2, c / 2, cs);
  S* const kd = static_cast<S*>(p.c.kc) + page * p.c.skc[0] + in * p.c.skc[1] + c;
  S* const vd = static_cast<S*>(p.c.vc) + page * p.c.svc[0] + in * p.c.svc[1] + c;
#pragma unroll
  for (int i = 0; i < kAppendHeads; ++i) {
    if (h0 + i >= p.Hkv) break;
    rope_rotate8(x[i], cs);
    put_row8<S>(kd + (h0 + i) * p.c.skc[2], x[i]);
    *reinterpret_cast<Raw8<S>*>(vd + (h0 + i) * p.c.svc[2]) = v[i];
  }
}

template <typename S, int D>
static hipError_t append(const AppendParams& p, hipStream_t st) {
  const int rows = 256 / (D / 8), n_grp = (p.Hkv + kAppendHeads - 1) / kAppendHeads;
  const int n_blk = (p.T + rows - 1) / rows;
  hipLaunchKernelGGL((cache_append_kernel<S, D>), dim3(n_blk * n_grp), dim3(256), 0, st, p, n_grp);
  return hipGetLastError();
}
template <typename S>
static hipError_t append_d(const AppendParams& p, int D, hipStream_t st) {
  return D == 32 ? append<S, 32>(p, st) : D == 64 ? append<S, 64>(p, st) : D == 128 ? append<S, 128>(p, st) : append<S, 256>(p, st);
}
hipError_t launch_cache_append(const AppendParams& p, int dt, int D, hipStream_t st) {
  return dt == DT_BF16 ? append_d<bf16>(p, D, st) : dt == DT_F16 ? append_d<f16>(p, D, st) : append_d<float>(p, D, st);
}

}  // namespace farope
