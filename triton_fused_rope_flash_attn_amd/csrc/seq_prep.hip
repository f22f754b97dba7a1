// Rotated key rows of packed sequences: what the forward's and the backward's
// tiles stream.
//
// K-hat = scale * log2(e) * R(position) K, rounded once to the tensors' type, as
// [Hkv, T, D]; and, where V's own rows cannot be streamed (channels not
// contiguous, or rows not 16-byte aligned), V copied to the same layout.  A
// thread takes 8 channels of one token and kPrepHeads key heads, so that their
// loads are in flight together and share one read of the table row.  The first
// workgroups also find the tiles of the slots that the kernels behind will take,
// one slot a wave.  Bound by memory: 11452 tokens, 12 heads, D 64 8.6 us (36 MB, 4.2 TB/s).
#include "seq.h"

namespace farope {

constexpr int kPrepHeads = 4;
struct SeqMaps {
  int slots_q, slots_k, lb_q;   // slots of the query and key kernels; rows of a query slot: 2^lb_q
  int blocks;                   // workgroups that fill the maps
  int order;                    // tiles in the order of their work
};

template <typename S, int D>
__global__ void __launch_bounds__(256) seq_prep_kernel(const SeqParams p, const SeqMaps m, int n_grp) {
  constexpr int CPR = D / 8, ROWS = 256 / CPR;
  const int tid = thread_id(), lane = tid & 63;
  if (block_id() < m.blocks) {
    int slot = 4 * block_id() + __builtin_amdgcn_readfirstlane(tid >> 6);
    const bool keys = slot >= m.slots_q;
    slot -= keys ? m.slots_q : 0;
    if (keys && slot >= m.slots_k) return;
    const int lb = keys ? 6 : m.lb_q;
    const SeqTile t = m.order ? ordered_tile(p.cu, p.B, p.T, lb, slot, lane, keys)
                              : find_tile(p.cu, p.B, p.T, lb, keys ? slot : m.slots_q - 1 - slot, lane);
    int* const to = (keys ? p.map_k : p.map_q) + 4 * (int64_t)slot;
    if (lane == 0) {
      to[0] = t.seq;
      to[1] = t.start;
      to[2] = t.len;
      to[3] = t.tile;
    }
    return;
  }
  const int id = block_id() - m.blocks, blk = id / n_grp, h0 = (id - blk * n_grp) * kPrepHeads;
  const int t0 = blk * ROWS, t = t0 + tid / CPR, c = 8 * (tid % CPR);
  const int tc = t < p.T ? t : p.T - 1;
  Raw8<S> k[kPrepHeads], v[kPrepHeads];   // (in flight while the token's sequence is found)
#pragma unroll
  for (int i = 0; i < kPrepHeads; ++i) {
    const int h = h0 + i < p.Hkv ? h0 + i : p.Hkv - 1;
    k[i] = load_raw8<S>(static_cast<const S*>(p.k) + tc * p.sk[0] + h * p.sk[1] + c * p.sk[2], p.sk[2], p.vec_k);
    if (p.vcopy) v[i] = load_raw8<S>(static_cast<const S*>(p.v) + tc * p.sv[0] + h * p.sv[1] + c * p.sv[2], p.sv[2], p.vec_v);
  }
  const int b = find_seq(p.cu, p.B, p.T, t0, tc, lane);
  if (t >= p.T || b == p.B) return;   // (no tile reads tokens of no sequence)
  const int row = table_row(p.positions ? p.positions[t] : t - cu_at(p.cu, b, p.T) - p.has_cls, p.n_pos);
  float cs[8];
  table_load4(p.cosp, p.sinp, row, D / 2, c / 2, cs);
#pragma unroll
  for (int i = 0; i < kPrepHeads; ++i) {
    if (h0 + i >= p.Hkv) break;
    float x[8];
    unpack8(k[i], x);
    rope_rotate8(x, cs);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= p.c2;
    const int64_t at = ((int64_t)(h0 + i) * p.T + t) * D + c;
    put_row8<S>(static_cast<S*>(p.khat) + at, x);
    if (p.vcopy) *reinterpret_cast<Raw8<S>*>(static_cast<S*>(p.vcopy) + at) = v[i];
  }
}

template <typename S, int D>
static hipError_t prep(const SeqParams& p, bool backward, hipStream_t st) {
  SeqMaps m{};
  m.order = seq_order(p.T, p.B, D, p.causal, p.window);
  m.lb_q = seq_tile_rows(p.T, p.B, p.H, D, sizeof(S) == 4) == 128 ? 7 : 6;
  m.slots_q = (int)seq_slots(p.T, p.B, m.lb_q);
  m.slots_k = backward ? (int)seq_slots(p.T, p.B, 6) : 0;
  m.blocks = (m.slots_q + m.slots_k + 3) / 4;
  const int rows = 256 / (D / 8), n_grp = (p.Hkv + kPrepHeads - 1) / kPrepHeads;
  const int n_blk = (p.T + rows - 1) / rows;
  hipLaunchKernelGGL((seq_prep_kernel<S, D>), dim3((unsigned)m.blocks + (unsigned)n_blk * n_grp), dim3(256), 0, st, p, m, n_grp);
  return hipGetLastError();
}
template <typename S>
static hipError_t prep_d(const SeqParams& p, int D, bool b, hipStream_t st) {
  return D == 32 ? prep<S, 32>(p, b, st) : D == 64 ? prep<S, 64>(p, b, st) : D == 128 ? prep<S, 128>(p, b, st) : prep<S, 256>(p, b, st);
}
hipError_t launch_seq_prep(const SeqParams& p, int dt, int D, bool b, hipStream_t st) {
  return dt == DT_BF16 ? prep_d<bf16>(p, D, b, st) : dt == DT_F16 ? prep_d<f16>(p, D, b, st) : prep_d<float>(p, D, b, st);
}

}  // namespace farope
