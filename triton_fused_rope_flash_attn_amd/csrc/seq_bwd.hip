// Backward of attention over packed sequences, from O, dO and the forward's LSE:
//
//   P = exp(s - LSE), delta_i = dO_i.O_i, dS = P * (dO V^T - delta)
//   dV_j = sum_i P_ij dO_i             over the query heads of the key head
//   dQ_i = R^T scale sum_j dS_ij R k_j
//   dK_j = R^T scale sum_i dS_ij R q_i over the query heads of the key head
//
// Three launches (short sequences: the last two, which then rotate K themselves):
//   seq_prep_kernel   K-hat * c2 rows (c2 = scale * log2 e)
//   seq_dq_kernel     query tiles: dQ; also -delta, -LSE * log2 e and the rotated Q rows (fp16, D 128: dO's norms)
//   seq_dkdv_kernel   key tiles: dK, dV, one pass over the group's query heads, so the
//                     sums of shared key heads stay in registers and in one order
// With a window (WIN) a key tile's queries end with its last key's window, but for tiles with sinks, whose queries
// are divided (KeyTile), joined by sink_join_kernel and taken in an order of their own (QueryStages); and rows that see 64 keys at most,
// which may be anywhere, have their delta from a pass of its own over the tile's keys (two of its four products).  One of 16384
// tokens, 8 heads, 2 of keys, D 128, 4 sinks, window 1024: dQ 163 us, dK/dV 216; the whole step with window 20, all rows with that
// pass, 213, with 64, none but the first tile's, 203.
// Both tile kernels stream their rows as the forward does (seq_fwd.hip).  No row of a
// sequence reads another's: streams end at the sequence's last row.
//
// Bound as the forward is.  One sequence of 16384 tokens, 8 heads (2 of keys), D 128, causal: dQ
// 750 us for its three products (1100 TFLOP/s), dK/dV 1230 for its four (895 TFLOP/s); 64
// sequences up to 577, 12 heads, D 64: 41 and 43 us, of which waves wait 66% and 53%.
#include <type_traits>

#include "seq.h"

namespace farope {

// Where a logit's -LSE2 (and dP's -delta) enters its sum: with 16-bit operands as the
// accumulator's start; with fp32 ones at the end, so that the partial sums do not round
// at LSE's size (dV at D 128, up to 577 tokens: off by 5.7e-7 of its norm, 1.6e-6 otherwise).
template <typename S> __device__ __forceinline__ f32x4 first_sum(f32x4 x) { return sizeof(S) == 4 ? f32x4{0.f, 0.f, 0.f, 0.f} : x; }
template <typename S> __device__ __forceinline__ void last_sum(f32x4& acc, f32x4 x) {
  if constexpr (sizeof(S) == 4) acc += x;
}

// fp16's normal values end at 2^-14 and its largest is 65504, while dS = P (dP - delta) of a row
// of n keys is about |dO| |V| / n.  There the products take 2^ex dS, rounded once, with a power of two that
// follows the values: where one passes the range, ex goes down and the sums held so far with it; the sums'
// last factor takes it out (all of it exact).  Without (4096 tokens, D 128) a dO of 1e-4 left dQ and dK
// off by 1.1e-2 of their norm, where rounding the exact ones to fp16 costs 2.7e-3 and 1.9e-3 (with: 2.8e-3
// and 2.0e-3), and a dP past 65504 made them NaN.  Forward and backward take 0 to 6% longer for it (us, 24
// up to 2048, 16 heads, D 128 858 / 880, 64 up to 577, 12 heads, D 64 153 / 158, 2 x 4096, 8 heads, D 256 1169 /
// 1236).  bf16 has fp32's exponents and needs none.
template <typename S> constexpr bool kFitDs = std::is_same<S, f16>::value;
constexpr float kDsMost = 32768.f;
constexpr int kExMost = 60, kExLeast = -100;
__device__ __forceinline__ float pow2(int e) { return __builtin_amdgcn_ldexpf(1.f, e); }
// The exponent that puts m >= 0 into [2^top, 2 * 2^top).
__device__ __forceinline__ int fit_exponent(float m, int top) {
  const int e = top + 127 - (int)(__float_as_uint(m) >> 23);
  return e > kExMost ? kExMost : e < kExLeast ? kExLeast : e;
}
// |x|, or 0 where it is infinite or NaN (which no scale helps, and which must not take the others')
__device__ __forceinline__ float finite_size(float x) {
  const unsigned u = magnitude_bits(x);
  return u < kInfBits ? __uint_as_float(u) : 0.f;
}

// Gradient rows of a 16-row subtile: lane holds row `row` (byte offset off), channels
// c0 + 16d + 4lg + (0..3) of each acc[d]; rows past the range of r drop.  turn: rotated back by
// the row of its token.
template <typename S, int D, int N>
__device__ __forceinline__ void store_tiles(const f32x4 (&acc)[N], int c0, float factor, bool turn, const SeqParams& p, int table,
                                            __amdgpu_buffer_rsrc_t r, unsigned off, int lg) {
  f32x4 g[N];
#pragma unroll
  for (int d = 0; d < N; ++d) {
    g[d] = acc[d] * factor;
    if (turn && table >= 0) {
      typedef float f2 __attribute__((ext_vector_type(2)));
      const int64_t at = (int64_t)table * (D / 2) + c0 / 2 + 8 * d + 2 * lg;
      const f2 c = *reinterpret_cast<const f2*>(p.cosp + at), s = *reinterpret_cast<const f2*>(p.sinp + at);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float e = g[d][2 * k], o = g[d][2 * k + 1];
        g[d][2 * k] = e * c[k] + o * s[k];
        g[d][2 * k + 1] = o * c[k] - e * s[k];
      }
    }
  }
  if constexpr (sizeof(S) == 4) {
#pragma unroll
    for (int d = 0; d < N; ++d) buf_store16(__builtin_bit_cast(u32x4, g[d]), r, off + (unsigned)(c0 + 16 * d + 4 * lg) * 4u, 0u);
  } else {
    u32x2 w[N];
#pragma unroll
    for (int d = 0; d < N; ++d) {
      typedef S s4 __attribute__((ext_vector_type(4)));
      s4 a;
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] = (S)g[d][e];
      __builtin_memcpy(&w[d], &a, 8);
    }
    if constexpr (N % 2) {
#pragma unroll
      for (int d = 0; d < N; ++d)
        __builtin_amdgcn_raw_buffer_store_b64(w[d], r, off + (unsigned)(c0 + 16 * d + 4 * lg) * 2u, 0u, 0);
    } else {
      // lane groups lg and lg^1 trade halves so that each lane stores 8 consecutive channels
#pragma unroll
      for (int d0 = 0; d0 < N; d0 += 2) {
        u32x4 x;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const auto y = __builtin_amdgcn_permlane16_swap(w[d0][k], w[d0 + 1][k], false, false);
          x[k] = y[0];
          x[2 + k] = y[1];
        }
        buf_store16(x, r, off + (unsigned)(c0 + 16 * (d0 + (lg & 1)) + 4 * (lg & 2)) * 2u, 0u);
      }
    }
  }
}
template <typename S, int D>
__device__ __forceinline__ void store_rows(const f32x4 (&acc)[D / 16], float factor, bool turn, const SeqParams& p, int table,
                                           __amdgpu_buffer_rsrc_t r, unsigned off, int lg) {
  store_tiles<S, D, D / 16>(acc, 0, factor, turn, p, table, r, off, lg);
}

// rows of zeros: tokens behind the last sequence
template <typename S, int D>
__device__ __forceinline__ void zero_rows(S* base, int64_t stride, int rows, int tid) {
  for (int r = tid / (D / 8); r < rows; r += kSeqThreads / (D / 8)) {
    const float z[8] = {};
    put_row8<S>(base + (int64_t)r * stride + 8 * (tid % (D / 8)), z);
  }
}

// A window of one token and no sinks: every row sees itself alone.
template <bool WIN> __device__ __forceinline__ bool sees_itself(const SeqParams& p) { return WIN && p.window == 1 && p.sinks == 0; }
// What the sums dS^T Q-hat are multiplied by: a sequence of one token has dS = 0, which the sums,
// with -delta as their start, hold but for rounding.
template <bool WIN>
__device__ __forceinline__ float dk_factor(const SeqParams& p, int len) { return len == 1 || sees_itself<WIN>(p) ? 0.f : p.scale; }

// ---------------------------------------------------------------------------
// dQ of 64 QT query rows of one head.  S^T = K-hat Q-hat^T and dP^T = V dO^T per
// 32-key block; their output rows are the k-slots of dQ-hat^T += K-hat^T dS^T.
// ---------------------------------------------------------------------------
// Keys of a stage: as in the forward (short sequences: 64, so that one stage holds them).  Two stages hold 64 at least.
template <typename S, int D, bool ROT> constexpr int kDqRows = sizeof(S) == 2 && D == 128 && !ROT ? 32 : kStageRowsOf<S, D>;
template <typename S, int D, int QT, bool ROT, bool WIN>
__global__ void __launch_bounds__(kSeqThreads, (sizeof(S) == 4 || D == 256) ? 1 : D == 128 && (QT == 2 || ROT) ? 2 : 3)
seq_dq_kernel(const SeqParams p) {
  using C = typename SeqComp<S>::C;
  using Frag = typename C::Frag;
  using T = Tile<S, D, kDqRows<S, D, ROT>>;
  constexpr int KS = D / 32, DT = D / 16, SR = T::SR, NB = SR / 32, LB = QT == 2 ? 7 : 6;
  __shared__ __attribute__((aligned(16))) S sK0[SR * D], sK1[SR * D], sV0[SR * D], sV1[SR * D];

  const int tid = thread_id();
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int lr = lane & 15, lg = lane >> 4;
  const int slot = block_id() / p.H, hx = block_id() % p.H;   // (as in the forward)
  const int kvh = hx % p.Hkv, head = kvh * (p.H / p.Hkv) + hx / p.Hkv;
  const SeqTile tl = slot_tile(p, LB, slot, lane, false);
  if (tl.tile < 0) return;
  const int q0 = tl.tile << LB, rows = tl.len - q0 < (1 << LB) ? tl.len - q0 : 1 << LB;
  const int64_t tok0 = tl.start + q0;
  S* const dqb = static_cast<S*>(p.dq) + (tok0 * p.H + head) * D;
  if (tl.seq == p.B) {
    zero_rows<S, D>(dqb, (int64_t)p.H * D, rows, tid);
    return;
  }

  const KeyStages<WIN, SR> ks(p, q0, q0 + (1 << LB), tl.len);
  SeqStream<S, D, T::SR> srcK, srcV;
  RotStage<S, D, T::SR> rot;
  if constexpr (ROT) {
    rot.load(p, tl, kvh, ks.at(0), tid);
  } else {
    srcK.lanes(D, wave, lane);
    srcK.base(static_cast<const S*>(p.khat) + ((int64_t)kvh * p.T + tl.start) * D, tl.len);
    srcK.load(sK0, wave, ks.at(0) * SR);
  }
  if (!ROT && p.vcopy) {
    srcV.lanes(D, wave, lane);
    srcV.base(static_cast<const S*>(p.vcopy) + ((int64_t)kvh * p.T + tl.start) * D, tl.len);
  } else {
    srcV.lanes(p.sv[0], wave, lane);
    srcV.base(static_cast<const S*>(p.v) + tl.start * p.sv[0] + kvh * p.sv[1], tl.len);
  }
  srcV.load(sV0, wave, ks.at(0) * SR);

  const int row0 = wave * 16 * QT + lr;   // of the tile; subtile t: + 16 t
  const int64_t hrow = (int64_t)head * p.T + tok0;
  const int w0 = q0 + wave * 16 * QT;   // the wave's first row (uniform)
  const bool active = w0 < tl.len;
  const int lo = p.causal ? w0 + 1 : tl.len;
  const int hi = p.causal && w0 + 16 * QT < tl.len ? w0 + 16 * QT : tl.len;
  const int ns = ks.n;
  const bool few = !WIN && q0 == 0 && (p.causal || tl.len <= 64);   // some rows of the tile see 64 keys at most
  // (with a window: they may be anywhere, and have their delta from a pass of its own over the tile's keys)
  const bool twice = WIN && (q0 == 0 || p.window <= 64 - p.sinks);
  const bool mine = few && hi <= 64;                        // (uniform) and so do all of the wave's
  Frag qf[QT][KS], gf[QT][KS];
  f32x4 nl4[QT], nd4[QT];
  int seen[QT], trow[QT];
  int ex[QT];   // kFitDs: P, and with it dS, carries 2^ex of its row
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = row0 + 16 * t, rc = r < rows ? r : rows - 1;
    const int64_t tok = tok0 + rc;
    const S* qp = static_cast<const S*>(p.q) + tok * p.sq[0] + head * p.sq[1];
    const S* gp = static_cast<const S*>(p.dout) + tok * p.sdo[0] + head * p.sdo[1];
    const S* op = static_cast<const S*>(p.o) + (tok * p.H + head) * D;
    seen[t] = p.causal ? q0 + rc + 1 : tl.len;
    trow[t] = table_row(p.positions ? p.positions[tok] : q0 + rc - p.has_cls, p.n_pos);
    float ds = 0.f, most = 0.f, size = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int c = 32 * s + 8 * lg;
      float x[8], g[8], o[8], cs[8];
      load8<S>(qp + c * p.sq[2], p.sq[2], p.vec_q, x);
      load8<S>(gp + c * p.sdo[2], p.sdo[2], p.vec_do, g);
      load8<S>(op + c, 1, true, o);
      table_load4(p.cosp, p.sinp, trow[t], D / 2, c / 2, cs);
      rope_rotate8(x, cs);
      qf[t][s] = C::make(x);
      gf[t][s] = C::make(g);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        ds += g[e] * o[e];
        if constexpr (kFitDs<S> && D == 128) size += g[e] * g[e];
      }
      if constexpr (kFitDs<S>) most = amax8(most, g);
      if (r < rows) {
        put_row8<S>(static_cast<S*>(p.qhat) + (hrow + r) * D + c, x);
        if (p.gcopy) put_row8<S>(static_cast<S*>(p.gcopy) + (hrow + r) * D + c, g);
      }
    }
    const float nd = -group4_sum(ds), nl = -p.lse[hrow + rc] * kLog2e;
    const float norm = kFitDs<S> && D == 128 ? __builtin_sqrtf(group4_sum(size)) : 0.f;
    if (r < rows && lg == 0) {
      p.nl[hrow + r] = nl + kWeightUp<S>;
      p.nd[hrow + r] = nd;
      if constexpr (kFitDs<S> && D == 128) p.ng[hrow + r] = norm;
    }
    // (at first the largest |dO| in [2^14, 2^15): dS is P |V| times that or a few times it)
    ex[t] = kFitDs<S> && !mine ? fit_exponent(group4_max(most), 14) : 0;
    const float nlx = nl + (float)ex[t];
    nl4[t] = f32x4{nlx, nlx, nlx, nlx};
    nd4[t] = f32x4{nd, nd, nd, nd};
  }

  f32x4 acc[QT][DT];
#pragma unroll
  for (int t = 0; t < QT; ++t)
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  FragAt<S, D> at;
  at.init(lr, lg);

  // key 16 h + i of the lane's part of a block is one that its row of the subtile sees; lim: those behind its keys
  auto sees = [&](int e, int lim, int k0) __attribute__((always_inline)) {
    return e < lim && (!WIN || e >= lim - p.window || e < p.sinks - k0 - 4 * lg);
  };
  auto block = [&](bool tail, bool edge, int k0, const S* __restrict__ k, const S* __restrict__ v) __attribute__((always_inline)) {
    f32x4 sacc[QT][2], pacc[QT][2];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const Frag a = at.row(k, s, h), b = at.row(v, s, h);
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          sacc[t][h] = C::mma(a, qf[t][s], s == 0 ? first_sum<S>(nl4[t]) : sacc[t][h]);
          pacc[t][h] = C::mma(b, gf[t][s], s == 0 ? first_sum<S>(nd4[t]) : pacc[t][h]);
          if (s == KS - 1) {
            last_sum<S>(sacc[t][h], nl4[t]);
            last_sum<S>(pacc[t][h], nd4[t]);
          }
        }
      }
    Frag dsf[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      // (a row that sees one key: P = 1, dS = 0)
      const int lim = (seen[t] > 1 && !sees_itself<WIN>(p) ? seen[t] : 0) - k0 - 4 * lg;
      float ds[8];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float y = fast_exp2(sacc[t][h][i]) * pacc[t][h][i];
          ds[4 * h + i] = !tail || 16 * h + i < lim ? y : 0.f;
        }
      if (WIN && edge) {
        const int from = seen[t] - p.window - k0 - 4 * lg, sinks = p.sinks - k0 - 4 * lg;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) ds[4 * h + i] = 16 * h + i >= from || 16 * h + i < sinks ? ds[4 * h + i] : 0.f;
      }
      if constexpr (kFitDs<S>) {
        const float most = amax8(0.f, ds);
        if (__any(most > kDsMost)) {   // rows that pass it start again from 2^12
          const float m = group4_max(most);
          const int down = m > kDsMost ? fit_exponent(m, 12) : 0;
          const float f = pow2(down);
          ex[t] += down;
          nl4[t] += (float)down;
#pragma unroll
          for (int e = 0; e < 8; ++e) ds[e] *= f;
#pragma unroll
          for (int d = 0; d < DT; ++d) acc[t][d] *= f;
        }
      }
      dsf[t] = C::make(ds);   // (16-bit tensors: dS rounded to their type for the product)
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const Frag a = at.col(k, d);
#pragma unroll
      for (int t = 0; t < QT; ++t) acc[t][d] = C::mma(a, dsf[t], acc[t][d]);
    }
  };
  // sum_j P_ij dP_ij of a block's keys (delta, in fp32)
  float sum[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) sum[t] = 0.f;
  auto sum_block = [&](int k0, const S* __restrict__ k, const S* __restrict__ v) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const int lim = seen[t] - k0 - 4 * lg;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f32x4 sacc, pacc;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          sacc = C::mma(at.row(k, s, h), qf[t][s], s == 0 ? first_sum<S>(nl4[t]) : sacc);
          pacc = C::mma(at.row(v, s, h), gf[t][s], s == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : pacc);
        }
        last_sum<S>(sacc, nl4[t]);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[t] += sees(16 * h + i, lim, k0) ? fast_exp2(sacc[i]) * pacc[i] : 0.f;
      }
    }
  };
  auto stage = [&](int st, bool sums, const S* __restrict__ k, const S* __restrict__ v, S* __restrict__ kn, S* __restrict__ vn)
      __attribute__((always_inline)) {
    seq_stage_barrier();
    if (st + 1 < ns) {
      if constexpr (ROT) rot.load(p, tl, kvh, ks.at(st + 1), tid);
      else srcK.load(kn, wave, ks.at(st + 1) * SR);
      srcV.load(vn, wave, ks.at(st + 1) * SR);
    }
    const int k0 = ks.at(st) * SR;
    if (active && k0 < hi && (!WIN || k0 + SR > w0 + 1 - p.window || k0 < p.sinks)) {
      const bool tail = k0 + SR > lo || sees_itself<WIN>(p), edge = WIN && past_window(p, k0, SR, hi - p.window);
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        if (WIN && sums) sum_block(k0 + 32 * j, k + 32 * j * D, v + 32 * j * D);
        else block(tail, edge, k0 + 32 * j, k + 32 * j * D, v + 32 * j * D);
      }
    }
    if (ROT && st + 1 < ns) rot.store(p, kn, tid);   // (read in the stage before this one)
  };
  if constexpr (ROT) rot.store(p, sK0, tid);
  // Rows that see 64 keys at most, all of them in LDS: delta = sum_j P_ij dP_ij, in fp32, while P and dP
  // are in registers.  Such rows have an O as large as V, whose rounding as stored would be the largest error
  // of a dS that cancels (sequences of two tokens, bf16: dQ off by 5e-3 of its norm from O dO; V of 64 + N(0, 1):
  // 0.16).  Key block j of 32 is at k[j], v[j].
  auto whole = [&](const S* const (&k)[2], const S* const (&v)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      f32x4 prob[2][2], pacc[2][2];
      const int lim = seen[t] - 4 * lg;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (32 * j >= hi) {   // (uniform: no such keys, and nothing in LDS)
#pragma unroll
          for (int h = 0; h < 2; ++h) prob[j][h] = pacc[j][h] = f32x4{0.f, 0.f, 0.f, 0.f};
          continue;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            prob[j][h] = C::mma(at.row(k[j], s, h), qf[t][s], s == 0 ? first_sum<S>(nl4[t]) : prob[j][h]);
            pacc[j][h] = C::mma(at.row(v[j], s, h), gf[t][s], s == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : pacc[j][h]);
          }
          last_sum<S>(prob[j][h], nl4[t]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool in = 32 * j + 16 * h + i < lim;
            prob[j][h][i] = in ? fast_exp2(prob[j][h][i]) : 0.f;
            sum += in ? prob[j][h][i] * pacc[j][h][i] : 0.f;
          }
        }
      }
      const float delta = group4_sum(sum);
      const int dlim = seen[t] > 1 ? lim : 0;   // (as in block)
      if (row0 + 16 * t < rows && lg == 0) p.nd[hrow + row0 + 16 * t] = -delta;
      float f = 1.f;
      if constexpr (kFitDs<S>) {
        float most = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              most = fmaxf(most, 32 * j + 16 * h + i < dlim ? fabsf(prob[j][h][i] * (pacc[j][h][i] - delta)) : 0.f);
        ex[t] = fit_exponent(group4_max(most), 14);
        f = pow2(ex[t]);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (32 * j >= hi) continue;
        float ds[8];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            ds[4 * h + i] = 32 * j + 16 * h + i < dlim ? prob[j][h][i] * (pacc[j][h][i] - delta) * f : 0.f;
        const Frag dsf = C::make(ds);
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[t][d] = C::mma(at.col(k[j], d), dsf, acc[t][d]);
      }
    }
  };
  int from = 0;
  if (few) {   // (uniform) the first two stages together
    if (ns > 1) {
      if constexpr (ROT) {
        rot.load(p, tl, kvh, 1, tid);
        rot.store(p, sK1, tid);
      } else {
        srcK.load(sK1, wave, SR);
      }
      srcV.load(sV1, wave, SR);
    }
    seq_stage_barrier();
    auto at_block = [&](const S* a, const S* b, int j) __attribute__((always_inline)) { return (j < NB ? a : b) + 32 * (j % NB) * D; };
    if (mine) {
      const S* const k[2] = {sK0, at_block(sK0, sK1, 1)};
      const S* const v[2] = {sV0, at_block(sV0, sV1, 1)};
      if (active) whole(k, v);
    } else if (active) {
#pragma unroll 1
      for (int j = 0; j < 2 * NB && 32 * j < hi; ++j) block(true, false, 32 * j, at_block(sK0, sK1, j), at_block(sV0, sV1, j));
    }
    from = 2;
    if (ns > 2) {
      lds_barrier();   // (all waves have read them)
      if constexpr (ROT) {
        rot.load(p, tl, kvh, 2, tid);
        rot.store(p, sK0, tid);
      } else {
        srcK.load(sK0, wave, 2 * SR);
      }
      srcV.load(sV0, wave, 2 * SR);
    }
  }
  if constexpr (WIN) {
    if (twice) {   // (uniform)
#pragma unroll 1
      for (int st = 0; st < ns; st += 2) {
        stage(st, true, sK0, sV0, sK1, sV1);
        if (st + 1 < ns) stage(st + 1, true, sK1, sV1, sK0, sV0);
      }
#pragma unroll
      for (int t = 0; t < QT; ++t) {   // (P carries 2^ex)
        const float nd = -group4_sum(sum[t]) * (kFitDs<S> ? pow2(-ex[t]) : 1.f);
        if (row0 + 16 * t < rows && lg == 0) p.nd[hrow + row0 + 16 * t] = nd;
        nd4[t] = f32x4{nd, nd, nd, nd};
      }
      lds_barrier();   // (all waves have read the last stages)
      if constexpr (ROT) {
        rot.load(p, tl, kvh, ks.at(0), tid);
        rot.store(p, sK0, tid);
      } else {
        srcK.load(sK0, wave, ks.at(0) * SR);
      }
      srcV.load(sV0, wave, ks.at(0) * SR);
    }
  }
  for (int st = from; st < ns; st += 2) {
    stage(st, false, sK0, sV0, sK1, sV1);
    if (st + 1 < ns) stage(st + 1, false, sK1, sV1, sK0, sV0);
  }

  const unsigned row_b = (unsigned)(p.H * D * (int)sizeof(S));
  const auto rD = make_rsrc(dqb, (unsigned)(rows - 1) * row_b + T::RB);
#pragma unroll
  for (int t = 0; t < QT; ++t)   // (K-hat carries scale * log2 e)
    store_rows<S, D>(acc[t], kFitDs<S> ? __builtin_amdgcn_ldexpf(kLn2, -ex[t]) : kLn2, true, p, trow[t], rD, (unsigned)(row0 + 16 * t) * row_b, lg);
}

// Queries from the returned one on do not see keys [first, last] (a key: first = last).
template <bool WIN>
__device__ __forceinline__ int key_reach(const SeqParams& p, int len, int first, int last) {
  return WIN && first >= p.sinks && len - last > p.window ? last + p.window : len;
}

// A workgroup's key tile, key head and part of the queries.  With a window all queries behind them see the sinks, so
// their tiles have many times the others' work: workgroups of the launch's end divide it into parts
// of their own, small ones that fill the chip while the last tiles are worked on, and the others leave it to them.
template <bool WIN> struct KeyTile {
  SeqTile tl;
  int part, parts, kvh;
  bool sinks;   // the sums go to p.spk and p.spv
  bool sums;
  __device__ __forceinline__ KeyTile(const SeqParams& p, int lane) {
    int id = block_id();
    sinks = false;
    if constexpr (WIN) {
      const int tiles = p.slots * p.Hkv * p.parts;
      if (id >= tiles) {
        id -= tiles;
        sinks = sums = true;
        parts = p.sink_parts;
        part = id % parts;
        id /= parts;
        kvh = id % p.Hkv;
        id /= p.Hkv;
        tl.tile = id % p.sink_tiles;
        tl.seq = id / p.sink_tiles;
        tl.start = cu_at(p.cu, tl.seq, p.T);
        const int end = cu_at(p.cu, tl.seq + 1, p.T);
        tl.len = end > tl.start ? end - tl.start : 0;
        tl.tiles = (tl.len + 63) >> 6;
        if (tl.tile >= tl.tiles) tl.tile = -1;
        return;
      }
    }
    parts = p.parts;
    sums = parts > 1;
    part = id % parts;
    id /= parts;
    kvh = id % p.Hkv;
    tl = slot_tile(p, 6, id / p.Hkv, lane, true);
    if (WIN && p.sink_parts && tl.seq < p.B && tl.tile < p.sink_tiles) tl.tile = -1;
  }
  // the first row of the sums (in rows of D)
  __device__ __forceinline__ int64_t sums_at(const SeqParams& p, int64_t tok0) const {
    if (sinks) return ((((int64_t)part * p.B + tl.seq) * p.sink_tiles + tl.tile) * 64) * p.Hkv + kvh;
    return ((int64_t)part * p.T + tok0) * p.Hkv + kvh;
  }
};

// The order of a key tile's stages of queries: head by head, the last queries first, as far back as the tile's first key when
// causal.  (Every tile of a sequence then begins with the same rows, which come from L2.  Measured (us, forward and backward,
// first / last queries first): 16 sequences up to 2048 tokens, 16 heads (4 of keys), D 64 406 / 390, 64 up to 577, 12
// 143 / 140, 8 x 1024, 8, D 128 159 / 156, one sequence of 16384 2510 / 2494 (HBM reads of the kernel 1716 / 419 MB).)
// With a window the far queries, which see of the tile's keys the sinks alone, come first in all heads: behind them the sums of
// the other keys, of weights that are 0, begin again from 0 (drop).  A query that is not finite, far from every query that sees such
// a key, so does not reach it as 0 * NaN.  (What this costs, us without / with, window 1024 or 512, 4 sinks, D 64 267 / 269, D 128 457 / 456,
// fp32 892 / 903, D 256 3635 / 3690, fp32 1858 / 1930: registers that the drop's results are moved through.)
template <bool WIN> struct QueryStages {
  int first, near, far;   // the first stage; stages of a head that are near (without a window: all) and far
  __device__ __forceinline__ QueryStages(const SeqParams& p, int k0, int len, int sr) {
    first = p.causal ? k0 / sr : 0;
    near = (key_reach<WIN>(p, len, k0, k0 + 63) + sr - 1) / sr - first;
    far = 0;
    if (WIN && k0 < p.sinks && k0 + 64 > p.sinks) {
      const int all = near;
      near = (key_reach<WIN>(p, len, p.sinks, k0 + 63) + sr - 1) / sr - first;
      far = all - near;
    }
  }
};

// ---------------------------------------------------------------------------
// dK and dV of 64 key rows of one key head.  Wave w owns 16 of them: their K-hat and
// V rows are operands in registers, dK-hat and dV accumulate in registers over the
// stages of every query head of the group (parts > 1: over a part's equal share of
// them).  128 keys per workgroup (D 32 and 64) measured the same within 3% for long
// sequences and slower for short ones (64 up to 577, D 64: 146 / 163 us).
// ---------------------------------------------------------------------------
template <typename S, int D, bool WIN>
__global__ void __launch_bounds__(kSeqThreads, (sizeof(S) == 4 || D == 256) ? 1 : 2) seq_dkdv_kernel(const SeqParams p) {
  using C = typename SeqComp<S>::C;
  using Frag = typename C::Frag;
  using T = Tile<S, D>;
  constexpr int KS = D / 32, DT = D / 16, SR = T::SR, NB = SR / 32, LB = 6;
  __shared__ __attribute__((aligned(16))) S sQ0[SR * D], sQ1[SR * D], sG0[SR * D], sG1[SR * D];
  __shared__ __attribute__((aligned(16))) float sL0[64], sL1[64], sD0[64], sD1[64];

  const int tid = thread_id();
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int lr = lane & 15, lg = lane >> 4;
  // earlier keys (seen by more queries) come first in each sequence
  const KeyTile<WIN> kt(p, lane);
  const int part = kt.part, parts = kt.parts, kvh = kt.kvh, group = p.H / p.Hkv;
  const SeqTile tl = kt.tl;
  if (tl.tile < 0) return;
  const int k0 = tl.tile << LB, rows = tl.len - k0 < (1 << LB) ? tl.len - k0 : 1 << LB;
  const int64_t tok0 = tl.start + k0;
  S* const dkb = static_cast<S*>(p.dk) + (tok0 * p.Hkv + kvh) * D;
  S* const dvb = static_cast<S*>(p.dv) + (tok0 * p.Hkv + kvh) * D;
  if (tl.seq == p.B) {
    if (parts > 1) return;   // (seq_join_kernel's)
    zero_rows<S, D>(dkb, (int64_t)p.Hkv * D, rows, tid);
    zero_rows<S, D>(dvb, (int64_t)p.Hkv * D, rows, tid);
    return;
  }

  // this part's share of all heads' stages, the far ones first; `run` of a head, the last of them `top`
  const QueryStages<WIN> qs(p, k0, tl.len, SR);
  const int64_t all = (int64_t)(qs.far + qs.near) * group;
  const int begin = (int)(all * part / parts), end = (int)(all * (part + 1) / parts);
  const bool far = WIN && begin < qs.far * group;
  const int begin_in = WIN && !far ? begin - qs.far * group : begin;   // among the far or near ones
  int run = far ? qs.far : qs.near, top = qs.first + (far ? qs.far + qs.near : qs.near) - 1;
  // Stages are numbered from `odd`, 0 or 1, on, so that the first near one behind far ones, `turn`, is even.
  const int odd = far ? (qs.far * group - begin) & 1 : 0, turn = far ? qs.far * group - begin + odd : 0, ns = end - begin + odd;
  SeqStream<S, D> srcQ, srcG;
  srcQ.lanes(D, wave, lane);
  srcG.lanes(p.gcopy ? D : p.sdo[0], wave, lane);
  int lh = begin_in / run - 1, lst = run, cst = begin_in % run;   // the stage loaded next: head of the group, stage
  int from = cst;
  __amdgpu_buffer_rsrc_t rStat = make_rsrc(p.nl, 0u);
  // (at `turn` the stage before it has been loaded)
  auto load = [&](S* q, S* g, float* l, float* d) __attribute__((always_inline)) {
    if (lst == run) {
      lst = from;
      from = 0;
      const int head = kvh * group + ++lh;
      const int64_t hrow = (int64_t)head * p.T + tl.start;
      srcQ.base(static_cast<const S*>(p.qhat) + hrow * D, tl.len);
      srcG.base(p.gcopy ? static_cast<const S*>(p.gcopy) + hrow * D
                        : static_cast<const S*>(p.dout) + tl.start * p.sdo[0] + head * p.sdo[1], tl.len);
      rStat = make_rsrc((wave & 1 ? p.nd : p.nl) + hrow, (unsigned)tl.len * 4u);
    }
    const int r0 = (top - lst) * SR;
    srcQ.load(q, wave, r0);
    srcG.load(g, wave, r0);
    // waves 0 and 1 also fetch the stage's -LSE2 and -delta (64 rows, of which SR count)
    if (wave < 2) seq_dma4(rStat, wave ? d : l, (unsigned)lane * 4u, (unsigned)r0 * 4u);
    ++lst;
  };
  if (end > begin) {
    if (WIN && odd) load(sQ1, sG1, sL1, sD1);
    else load(sQ0, sG0, sL0, sD0);
  }

  const int row0 = wave * 16 + lr;   // of the tile
  Frag kf[KS], vf[KS];
  const int rc = row0 < rows ? row0 : rows - 1;
  const int64_t tok = tok0 + rc;
  const S* const vp = static_cast<const S*>(p.v) + tok * p.sv[0] + kvh * p.sv[1];
  const int trow = table_row(p.positions ? p.positions[tok] : k0 + rc - p.has_cls, p.n_pos);
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const int c = 32 * s + 8 * lg;
    float x[8];
    if (p.khat) {
      load8<S>(static_cast<const S*>(p.khat) + ((int64_t)kvh * p.T + tok) * D + c, 1, true, x);
    } else {
      float cs[8];
      load8<S>(static_cast<const S*>(p.k) + tok * p.sk[0] + kvh * p.sk[1] + c * p.sk[2], p.sk[2], p.vec_k, x);
      table_load4(p.cosp, p.sinp, trow, D / 2, c / 2, cs);
      rope_rotate8(x, cs);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= p.c2;
    }
    kf[s] = C::make(x);
    load8<S>(vp + c * p.sv[2], p.sv[2], p.vec_v, x);
    vf[s] = C::make(x);
  }
  const int w0 = k0 + wave * 16;   // the wave's first key (uniform)
  const bool active = w0 < tl.len;
  // queries from here on do not see the lane's key, some of the wave's keys, any of them
  const int qend = key_reach<WIN>(p, tl.len, k0 + row0, k0 + row0);
  const int qfull = WIN ? w0 + 16 <= p.sinks ? tl.len : key_reach<WIN>(p, tl.len, p.sinks > w0 ? p.sinks : w0, w0) : tl.len;
  const int qlast = key_reach<WIN>(p, tl.len, w0, w0 + 15);
  f32x4 dv[DT], dk[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) dv[d] = dk[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  int ex = kFitDs<S> ? kExMost : 0;   // the wave's dS and dK carry 2^ex
  float fit = pow2(ex);
  FragAt<S, D> at;
  at.init(lr, lg);

  // 32 queries from q0 on; tail: some of them do not exist or do not see all of the wave's keys
  auto block = [&](bool tail, int q0, const S* __restrict__ q, const S* __restrict__ g, const float* __restrict__ l,
                   const float* __restrict__ dl) __attribute__((always_inline)) {
    f32x4 sacc[2], pacc[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 nl = *reinterpret_cast<const f32x4*>(l + 16 * h + 4 * lg);
      const f32x4 nd = *reinterpret_cast<const f32x4*>(dl + 16 * h + 4 * lg);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const Frag a = at.row(q, s, h), b = at.row(g, s, h);
        sacc[h] = C::mma(a, kf[s], s == 0 ? first_sum<S>(nl) : sacc[h]);
        pacc[h] = C::mma(b, vf[s], s == 0 ? first_sum<S>(nd) : pacc[h]);
      }
      last_sum<S>(sacc[h], nl);
      last_sum<S>(pacc[h], nd);
    }
    // query q0 + 16 h + 4 lg + i exists and sees this lane's key
    const int from = p.causal ? k0 + row0 - q0 - 4 * lg : -4 * lg, to = qend - q0 - 4 * lg;
    float pv[8], ds[8];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in = !tail || (16 * h + i >= from && 16 * h + i < to);
        const float e = fast_exp2(sacc[h][i]);
        pv[4 * h + i] = in ? e : 0.f;
        ds[4 * h + i] = in ? e * pacc[h][i] : 0.f;
      }
    if constexpr (kFitDs<S>) {
      const float most = amax8(0.f, ds) * fit;
      if (__any(most > kDsMost)) {
        float m = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fmaxf(m, finite_size(ds[e]));
        const int to = fit_exponent(__uint_as_float(__builtin_amdgcn_readfirstlane(wave_max_bits(m))), 12);
        if (to < ex) {
          const float f = pow2(to - ex);
#pragma unroll
          for (int d = 0; d < DT; ++d) dk[d] *= f;
          ex = to;
          fit = pow2(ex);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) ds[e] *= fit;
    }
    const Frag pf = C::make(pv), dsf = C::make(ds);   // (16-bit tensors: P and dS rounded to their type for the products)
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      dv[d] = C::mma(at.col(g, d), pf, dv[d]);
      dk[d] = C::mma(at.col(q, d), dsf, dk[d]);
    }
  };
  auto drop = [&]() __attribute__((always_inline)) {   // the sums of the lane's key, if it is no sink
    const bool sink = k0 + row0 < p.sinks;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        dv[d][i] = sink ? dv[d][i] : 0.f;
        dk[d][i] = sink ? dk[d][i] : 0.f;
      }
  };
  // (cst: this stage within its head)
  auto stage = [&](int st, const S* __restrict__ q, const S* __restrict__ g, const float* __restrict__ l, const float* __restrict__ dl,
                   S* __restrict__ qn, S* __restrict__ gn, float* __restrict__ ln, float* __restrict__ dn) __attribute__((always_inline)) {
    seq_stage_barrier();
    const int q0 = (top - cst) * SR;
    cst = cst + 1 == run ? 0 : cst + 1;
    if (WIN && st + 1 == turn) {   // (cst is 0, lst run)
      run = lst = qs.near;
      top = qs.first + qs.near - 1;
      lh = -1;
    }
    if (st + 1 < ns) load(qn, gn, ln, dn);
    if (!active || (p.causal && q0 + SR <= w0) || (WIN && q0 >= qlast)) return;
    const bool tail = q0 + SR > qfull || (p.causal && q0 < w0 + 16);
#pragma unroll
    for (int j = 0; j < NB; ++j)
      block(tail, q0 + 32 * j, q + 32 * j * D, g + 32 * j * D, l + 32 * j, dl + 32 * j);
  };
  for (int st = 0; st < ns; st += 2) {
    if (far && st == turn) drop();
    if (!WIN || st >= odd) stage(st, sQ0, sG0, sL0, sD0, sQ1, sG1, sL1, sD1);
    if (st + 1 < ns) stage(st + 1, sQ1, sG1, sL1, sD1, sQ0, sG0, sL0, sD0);
  }
  if (far && turn >= ns) drop();

  const float up = pow2(-(int)kWeightUp<S>);   // out of P
  if (kt.sums) {   // sums as they are, for seq_join_kernel
    const int64_t at = kt.sums_at(p, tok0) * D;
    const unsigned row_b = (unsigned)(p.Hkv * D) * 4u, bytes = (unsigned)(rows - 1) * row_b + D * 4u;
    const auto rpK = make_rsrc((kt.sinks ? p.spk : p.pk) + at, bytes), rpV = make_rsrc((kt.sinks ? p.spv : p.pv) + at, bytes);
    store_rows<float, D>(dk, pow2(-ex) * up, false, p, 0, rpK, (unsigned)row0 * row_b, lg);
    store_rows<float, D>(dv, up, false, p, 0, rpV, (unsigned)row0 * row_b, lg);
    return;
  }
  const unsigned row_b = (unsigned)(p.Hkv * D * (int)sizeof(S));
  const unsigned bytes = (unsigned)(rows - 1) * row_b + T::RB;
  const auto rdK = make_rsrc(dkb, bytes), rdV = make_rsrc(dvb, bytes);
  store_rows<S, D>(dk, dk_factor<WIN>(p, tl.len) * pow2(-ex) * up, true, p, trow, rdK, (unsigned)row0 * row_b, lg);
  store_rows<S, D>(dv, up, false, p, trow, rdV, (unsigned)row0 * row_b, lg);
}

// ---------------------------------------------------------------------------
// The same for 16-bit tensors at head_dim 128, bound otherwise by the LDS reads of waves
// that each need every query and dO row of a stage, both as rows and as columns.
// Here wave w takes one half of a stage's 64 queries against one half of the 64 keys
// (whose K-hat and V rows are operands in its registers) and leaves P and dS in LDS; then
// it takes its 32 channels of dV^T += dO^T P and dK-hat^T += Q-hat^T dS.  P and dS lie in
// LDS as the operands of those products.  LDS read per stage and wave: 40 KB instead of 64.
// Measured (us, forward and backward, seq_dkdv_kernel / this): 16384 tokens, 2 key heads
// 2696 / 2567, 24 up to 2048, 4 key heads 1094 / 1020, 8 x 4096, 8 1580 / 1501; at D 64 it is the
// slower one (8192, 16 key heads 717 / 742).
// ---------------------------------------------------------------------------
template <typename S, bool WIN>
__global__ void __launch_bounds__(kSeqThreads, 2) seq_dkdv_shared_kernel(const SeqParams p) {
  constexpr int D = 128;
  using C = typename SeqComp<S>::C;
  using Frag = typename C::Frag;
  using T = Tile<S, D>;
  constexpr int KS = D / 32, SR = T::SR, LB = 6, ND = D / 16 / kSeqNW;   // (ND: 16-channel tiles of a wave)
  static_assert(SR == 64 && sizeof(S) == 2, "");
  __shared__ __attribute__((aligned(16))) S sQ0[SR * D], sQ1[SR * D], sG0[SR * D], sG1[SR * D];
  __shared__ __attribute__((aligned(16))) S sP[2 * 4 * 64 * 8], sS[2 * 4 * 64 * 8];   // [block][subtile][lane][slot]

  const int tid = thread_id();
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int lr = lane & 15, lg = lane >> 4;
  const KeyTile<WIN> kt(p, lane);
  const int part = kt.part, parts = kt.parts, kvh = kt.kvh, group = p.H / p.Hkv;
  const SeqTile tl = kt.tl;
  if (tl.tile < 0) return;
  const int k0 = tl.tile << LB, rows = tl.len - k0 < (1 << LB) ? tl.len - k0 : 1 << LB;
  const int64_t tok0 = tl.start + k0;
  S* const dkb = static_cast<S*>(p.dk) + (tok0 * p.Hkv + kvh) * D;
  S* const dvb = static_cast<S*>(p.dv) + (tok0 * p.Hkv + kvh) * D;
  if (tl.seq == p.B) {
    if (parts > 1) return;   // (seq_join_kernel's)
    zero_rows<S, D>(dkb, (int64_t)p.Hkv * D, rows, tid);
    zero_rows<S, D>(dvb, (int64_t)p.Hkv * D, rows, tid);
    return;
  }

  // this part's share of all heads' stages, the far ones first; `run` of a head, the last of them `top`
  const QueryStages<WIN> qs(p, k0, tl.len, SR);
  const int64_t all = (int64_t)(qs.far + qs.near) * group;
  const int begin = (int)(all * part / parts), end = (int)(all * (part + 1) / parts);
  const bool far = WIN && begin < qs.far * group;
  const int begin_in = WIN && !far ? begin - qs.far * group : begin;   // among the far or near ones
  int run = far ? qs.far : qs.near, top = qs.first + (far ? qs.far + qs.near : qs.near) - 1;
  // Stages are numbered from `odd`, 0 or 1, on, so that the first near one behind far ones, `turn`, is even.
  const int odd = far ? (qs.far * group - begin) & 1 : 0, turn = far ? qs.far * group - begin + odd : 0, ns = end - begin + odd;
  SeqStream<S, D> srcQ, srcG;
  srcQ.lanes(D, wave, lane);
  srcG.lanes(p.gcopy ? D : p.sdo[0], wave, lane);
  int head = kvh * group + begin_in / run - 1, lst = run, cst = begin_in % run;   // of the stage loaded next
  int from = cst;
  __amdgpu_buffer_rsrc_t rNl = make_rsrc(p.nl, 0u), rNd = make_rsrc(p.nd, 0u), rNg = make_rsrc(p.nd, 0u);
  const int qh = wave & 1, kh = wave >> 1;   // the wave's halves of the queries and keys
  u32x4 nl_next[2], nd_next[2];              // -LSE2 and -delta of queries 32 qh + 16 h + 4 lg + (0..3)
  unsigned ng_next = 0, na_next = 0;         // kFitDs: |dO| and -delta of query `lane`
  auto load = [&](S* q, S* g) __attribute__((always_inline)) {
    if (lst == run) {
      lst = from;
      from = 0;
      ++head;
      const int64_t hrow = (int64_t)head * p.T + tl.start;
      srcQ.base(static_cast<const S*>(p.qhat) + hrow * D, tl.len);
      srcG.base(p.gcopy ? static_cast<const S*>(p.gcopy) + hrow * D
                        : static_cast<const S*>(p.dout) + tl.start * p.sdo[0] + head * p.sdo[1], tl.len);
      rNl = make_rsrc(p.nl + hrow, (unsigned)tl.len * 4u);
      rNd = make_rsrc(p.nd + hrow, (unsigned)tl.len * 4u);
      if constexpr (kFitDs<S>) rNg = make_rsrc(p.ng + hrow, (unsigned)tl.len * 4u);
    }
    const int r0 = (top - lst) * SR;
    srcQ.load(q, wave, r0);
    srcG.load(g, wave, r0);
    if constexpr (kFitDs<S>) {
      ng_next = __builtin_amdgcn_raw_buffer_load_b32(rNg, (unsigned)(r0 + lane) * 4u, 0u, 0);
      na_next = __builtin_amdgcn_raw_buffer_load_b32(rNd, (unsigned)(r0 + lane) * 4u, 0u, 0);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned at = (unsigned)(r0 + 32 * qh + 16 * h + 4 * lg) * 4u;
      nl_next[h] = __builtin_amdgcn_raw_buffer_load_b128(rNl, at, 0u, 0);
      nd_next[h] = __builtin_amdgcn_raw_buffer_load_b128(rNd, at, 0u, 0);
    }
    ++lst;
  };
  if (end > begin) {
    if (WIN && odd) load(sQ1, sG1);
    else load(sQ0, sG0);
  }

  Frag kf[2][KS], vf[2][KS];   // key 32 kh + 16 u + lr
  float vmax = 0.f;            // kFitDs: the largest |V_j| of the tile
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    float size = 0.f;
    const int r = 32 * kh + 16 * u + lr, rc = r < rows ? r : rows - 1;
    const int64_t tok = tok0 + rc;
    const S* const vp = static_cast<const S*>(p.v) + tok * p.sv[0] + kvh * p.sv[1];
    const int trow = p.khat ? 0 : table_row(p.positions ? p.positions[tok] : k0 + rc - p.has_cls, p.n_pos);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int c = 32 * s + 8 * lg;
      float x[8];
      if (p.khat) {
        load8<S>(static_cast<const S*>(p.khat) + ((int64_t)kvh * p.T + tok) * D + c, 1, true, x);
      } else {
        float cs[8];
        load8<S>(static_cast<const S*>(p.k) + tok * p.sk[0] + kvh * p.sk[1] + c * p.sk[2], p.sk[2], p.vec_k, x);
        table_load4(p.cosp, p.sinp, trow, D / 2, c / 2, cs);
        rope_rotate8(x, cs);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= p.c2;
      }
      kf[u][s] = C::make(x);
      load8<S>(vp + c * p.sv[2], p.sv[2], p.vec_v, x);
      vf[u][s] = C::make(x);
      if constexpr (kFitDs<S>) {
#pragma unroll
        for (int e = 0; e < 8; ++e) size += x[e] * x[e];
      }
    }
    if constexpr (kFitDs<S>) vmax = fmaxf(vmax, finite_size(__builtin_sqrtf(group4_sum(size))));
  }
  // Every wave has to know the scale of the dS that it takes from the others, and LDS has no room for it
  // (two workgroups fill the CU's).  So all of them derive it from the same numbers: |dS_ij| = P_ij |dP_ij -
  // delta_i| <= |dO_i| max |V_j| + |delta_i|, over a stage's queries and the tile's keys.
  int ex = kFitDs<S> ? kExMost : 0;
  float fit = pow2(ex);
  if constexpr (kFitDs<S>) {   // (sP is written behind the next barrier)
    float* const share = reinterpret_cast<float*>(sP);
    const unsigned most = wave_max_bits(vmax);
    if (lane == 0) share[wave] = __uint_as_float(most);
    lds_barrier();
    vmax = fmaxf(fmaxf(share[0], share[1]), fmaxf(share[2], share[3]));
  }
  f32x4 dv[4][ND], dk[4][ND];
#pragma unroll
  for (int u = 0; u < 4; ++u)
#pragma unroll
    for (int d = 0; d < ND; ++d) dv[u][d] = dk[u][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  FragAt<S, D> at;
  at.init(lr, lg);
  const int d0 = wave * ND;
  int to[ND];   // column reads of the wave's channels
#pragma unroll
  for (int d = 0; d < ND; ++d) to[d] = T::at(4 * lg + (lr >> 2), 16 * (d0 + d) + 4 * (lr & 3));
  const int qrow = 32 * qh * D;
  const int pw = ((4 * qh + 2 * kh) * 64 + lane) * 8;   // where the lane leaves its P and dS (subtile u, half h: + 512 u + 4 h)

  int qend[2];   // queries from here on do not see the lane's key
#pragma unroll
  for (int u = 0; u < 2; ++u) qend[u] = key_reach<WIN>(p, tl.len, k0 + 32 * kh + 16 * u + lr, k0 + 32 * kh + 16 * u + lr);
  // ... some of the tile's keys
  const int qfull = WIN ? k0 + 64 <= p.sinks ? tl.len : key_reach<WIN>(p, tl.len, p.sinks > k0 ? p.sinks : k0, k0) : tl.len;
  auto drop = [&]() __attribute__((always_inline)) {   // the sums of keys that are no sinks
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool sink = k0 + 16 * u + lr < p.sinks;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          dv[u][d][i] = sink ? dv[u][d][i] : 0.f;
          dk[u][d][i] = sink ? dk[u][d][i] : 0.f;
        }
    }
  };
  // (cst: this stage within its head)
  auto stage = [&](int st, const S* __restrict__ q, const S* __restrict__ g, S* __restrict__ qn, S* __restrict__ gn)
      __attribute__((always_inline)) {
    seq_stage_barrier();
    f32x4 nl[2], nd[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      nl[h] = __builtin_bit_cast(f32x4, nl_next[h]);
      nd[h] = __builtin_bit_cast(f32x4, nd_next[h]);
    }
    if constexpr (kFitDs<S>) {
      const float bound = finite_size(__uint_as_float(ng_next)) * vmax + finite_size(__uint_as_float(na_next));
      const int to = fit_exponent(__uint_as_float(__builtin_amdgcn_readfirstlane(wave_max_bits(finite_size(bound)))), 14 - (int)kWeightUp<S>);
      if (to < ex) {   // (uniform)
        const float f = pow2(to - ex);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int d = 0; d < ND; ++d) dk[u][d] *= f;
        ex = to;
        fit = pow2(ex);
      }
    }
    const int q0 = (top - cst) * SR;
    cst = cst + 1 == run ? 0 : cst + 1;
    if (WIN && st + 1 == turn) {   // (cst is 0, lst run)
      run = lst = qs.near;
      top = qs.first + qs.near - 1;
      head = kvh * group - 1;
    }
    if (st + 1 < ns) load(qn, gn);
    const bool tail = q0 + SR > qfull || (p.causal && q0 < k0 + 64);   // uniform
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      f32x4 sacc[2], pacc[2];
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const Frag a = C::lds(q + qrow + 16 * h * D + at.ao[s]), b = C::lds(g + qrow + 16 * h * D + at.ao[s]);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          sacc[u] = C::mma(a, kf[u][s], s == 0 ? nl[h] : sacc[u]);
          pacc[u] = C::mma(b, vf[u][s], s == 0 ? nd[h] : pacc[u]);
        }
      }
      // query qi + i (of the sequence) exists and sees key k0 + 32 kh + 16 u + lr
      const int qi = q0 + 32 * qh + 16 * h + 4 * lg, from = p.causal ? k0 + 32 * kh + lr - qi : -64;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        typedef S s4 __attribute__((ext_vector_type(4)));
        s4 pv, ds;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = !tail || (i >= from + 16 * u && i < qend[u] - qi);
          const float e = fast_exp2(sacc[u][i]);
          pv[i] = (S)(in ? e : 0.f);    // (P and dS rounded to the tensors' type for the products)
          ds[i] = (S)(in ? kFitDs<S> ? e * pacc[u][i] * fit : e * pacc[u][i] : 0.f);
        }
        *reinterpret_cast<s4*>(sP + pw + 512 * u + 4 * h) = pv;
        *reinterpret_cast<s4*>(sS + pw + 512 * u + 4 * h) = ds;
      }
    }
    lds_barrier();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      Frag ag[ND], aq[ND];
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        ag[d] = C::tr(g + 32 * j * D + to[d], g + 32 * j * D + to[d] + 16 * D);
        aq[d] = C::tr(q + 32 * j * D + to[d], q + 32 * j * D + to[d] + 16 * D);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int o = ((4 * j + u) * 64 + lane) * 8;
        const Frag pf = C::lds(sP + o), dsf = C::lds(sS + o);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          dv[u][d] = C::mma(ag[d], pf, dv[u][d]);
          dk[u][d] = C::mma(aq[d], dsf, dk[u][d]);
        }
      }
    }
  };
  for (int st = 0; st < ns; st += 2) {
    if (far && st == turn) drop();
    if (!WIN || st >= odd) stage(st, sQ0, sG0, sQ1, sG1);
    if (st + 1 < ns) stage(st + 1, sQ1, sG1, sQ0, sG0);
  }
  if (far && turn >= ns) drop();

  // lane holds key 16 u + lr, channels 16 (d0 + d) + 4lg + (0..3)
  const float up = pow2(-(int)kWeightUp<S>);   // out of P
  const unsigned es = kt.sums ? 4u : 2u, row_b = (unsigned)(p.Hkv * D) * es;
  const unsigned bytes = (unsigned)(rows - 1) * row_b + D * es;
  if (kt.sums) {   // sums as they are, for seq_join_kernel
    const int64_t w = kt.sums_at(p, tok0) * D;
    const auto rK = make_rsrc((kt.sinks ? p.spk : p.pk) + w, bytes), rV = make_rsrc((kt.sinks ? p.spv : p.pv) + w, bytes);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const unsigned off = (unsigned)(16 * u + lr) * row_b;
      store_tiles<float, D, ND>(dk[u], 16 * d0, pow2(-ex) * up, false, p, 0, rK, off, lg);
      store_tiles<float, D, ND>(dv[u], 16 * d0, up, false, p, 0, rV, off, lg);
    }
    return;
  }
  const auto rK = make_rsrc(dkb, bytes), rV = make_rsrc(dvb, bytes);
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int r = 16 * u + lr, rc = r < rows ? r : rows - 1;
    const int trow = table_row(p.positions ? p.positions[tok0 + rc] : k0 + rc - p.has_cls, p.n_pos);
    store_tiles<S, D, ND>(dk[u], 16 * d0, dk_factor<WIN>(p, tl.len) * pow2(-ex) * up, true, p, trow, rK, (unsigned)r * row_b, lg);
    store_tiles<S, D, ND>(dv[u], 16 * d0, up, false, p, trow, rV, (unsigned)r * row_b, lg);
  }
}

// dK and dV of the parts' sums, added in order; a thread takes 8 channels of one token
// and key head.
template <typename S, int D, bool WIN>
__global__ void __launch_bounds__(256) seq_join_kernel(const SeqParams p) {
  constexpr int CPR = D / 8, ROWS = 256 / CPR;
  const int blk = block_id() / p.Hkv, kvh = block_id() % p.Hkv;
  const int tid = thread_id(), t0 = blk * ROWS, t = t0 + tid / CPR, c = 8 * (tid % CPR);
  const int tc = t < p.T ? t : p.T - 1;
  const int b = find_seq(p.cu, p.B, p.T, t0, tc, tid & 63);
  if (t >= p.T) return;
  float k[8] = {}, v[8] = {};
  const int64_t at = ((int64_t)t * p.Hkv + kvh) * D + c;
  const int start = cu_at(p.cu, b, p.T);
  if (WIN && p.sink_parts && b < p.B && t - start < 64 * p.sink_tiles) return;   // (sink_join_kernel's)
  const int64_t step = (int64_t)p.T * p.Hkv * D;
  if (b < p.B) {
    for (int i = 0; i < p.parts; ++i) {
      float x[8], y[8];
      load8<float>(p.pk + i * step + at, 1, true, x);
      load8<float>(p.pv + i * step + at, 1, true, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) { k[e] += x[e]; v[e] += y[e]; }
    }
    const int row = table_row(p.positions ? p.positions[t] : t - start - p.has_cls, p.n_pos);
    const float factor = dk_factor<WIN>(p, cu_at(p.cu, b + 1, p.T) - start);
    float cs[8];
    table_load4(p.cosp, p.sinp, row, D / 2, c / 2, cs);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float e = k[2 * i] * factor, o = k[2 * i + 1] * factor;
      k[2 * i] = e * cs[2 * i] + o * cs[2 * i + 1];
      k[2 * i + 1] = o * cs[2 * i] - e * cs[2 * i + 1];
    }
  }
  put_row8<S>(static_cast<S*>(p.dk) + at, k);
  put_row8<S>(static_cast<S*>(p.dv) + at, v);
}

// The same of the tiles with sinks, whose parts are many: a workgroup takes one token and key head, its threads 8 channels
// of every so manieth part, and the threads' sums are added in order.
template <typename S, int D>
__global__ void __launch_bounds__(256) sink_join_kernel(const SeqParams p) {
  constexpr int CPR = D / 8, L = 256 / CPR;
  __shared__ __attribute__((aligned(16))) float sums[2][L][D];
  const int tid = thread_id(), c = 8 * (tid % CPR), l = tid / CPR;
  const int kvh = block_id() % p.Hkv, at = block_id() / p.Hkv, rows = 64 * p.sink_tiles, b = at / rows, j = at % rows;
  const int start = cu_at(p.cu, b, p.T), len = cu_at(p.cu, b + 1, p.T) - start;
  if (j >= len) return;
  float k[8] = {}, v[8] = {};
  const int64_t step = (int64_t)p.B * rows * p.Hkv * D, from = ((int64_t)at * p.Hkv + kvh) * D + c;
  for (int i = l; i < p.sink_parts; i += L) {
    float x[8], y[8];
    load8<float>(p.spk + i * step + from, 1, true, x);
    load8<float>(p.spv + i * step + from, 1, true, y);
#pragma unroll
    for (int e = 0; e < 8; ++e) { k[e] += x[e]; v[e] += y[e]; }
  }
  put_row8<float>(&sums[0][l][c], k);
  put_row8<float>(&sums[1][l][c], v);
  lds_barrier();
  if (l >= 2) return;
  float x[8] = {};
  for (int i = 0; i < L; ++i) {
    float y[8];
    load8<float>(&sums[l][i][c], 1, true, y);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] += y[e];
  }
  const int64_t t = start + j, to = (t * p.Hkv + kvh) * D + c;
  if (l == 0) {
    const float factor = dk_factor<true>(p, len);
    float cs[8];
    table_load4(p.cosp, p.sinp, table_row(p.positions ? p.positions[t] : j - p.has_cls, p.n_pos), D / 2, c / 2, cs);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float e = x[2 * i] * factor, o = x[2 * i + 1] * factor;
      x[2 * i] = e * cs[2 * i] + o * cs[2 * i + 1];
      x[2 * i + 1] = o * cs[2 * i] - e * cs[2 * i + 1];
    }
  }
  put_row8<S>(static_cast<S*>(l ? p.dv : p.dk) + to, x);
}

template <typename S, int D, int QT, bool ROT>
static hipError_t dq(const SeqParams& p0, hipStream_t st) {
  SeqParams p = p0;
  p.slots = (int)seq_slots(p.T, p.B, QT == 2 ? 7 : 6);
  const dim3 grid((unsigned)p.slots * p.H);
  if (p.window) hipLaunchKernelGGL((seq_dq_kernel<S, D, QT, ROT, true>), grid, dim3(kSeqThreads), 0, st, p);
  else hipLaunchKernelGGL((seq_dq_kernel<S, D, QT, ROT, false>), grid, dim3(kSeqThreads), 0, st, p);
  return hipGetLastError();
}
template <typename S, int D, bool WIN>
static hipError_t dkdv(const SeqParams& p, hipStream_t st) {
  const dim3 grid((unsigned)p.slots * p.Hkv * p.parts + (WIN ? (unsigned)p.B * p.sink_tiles * p.sink_parts * p.Hkv : 0u));
  if constexpr (sizeof(S) == 2 && D == 128)
    hipLaunchKernelGGL((seq_dkdv_shared_kernel<S, WIN>), grid, dim3(kSeqThreads), 0, st, p);
  else
    hipLaunchKernelGGL((seq_dkdv_kernel<S, D, WIN>), grid, dim3(kSeqThreads), 0, st, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  constexpr int rows = 256 / (D / 8);
  if (p.parts > 1)
    hipLaunchKernelGGL((seq_join_kernel<S, D, WIN>), dim3((unsigned)((p.T + rows - 1) / rows) * p.Hkv), dim3(256), 0, st, p);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  if constexpr (WIN)
    if (p.sink_parts)
      hipLaunchKernelGGL((sink_join_kernel<S, D>), dim3((unsigned)p.B * 64u * (unsigned)p.sink_tiles * p.Hkv), dim3(256), 0, st, p);
  return hipGetLastError();
}
template <typename S, int D>
static hipError_t bwd(const SeqParams& p0, hipStream_t st) {
  SeqParams p = p0;
  hipError_t e = hipSuccess;
  if (p.khat) {
    e = launch_seq_prep(p, std::is_same<S, bf16>::value ? DT_BF16 : std::is_same<S, f16>::value ? DT_F16 : DT_F32, D, true, st);
    if (e != hipSuccess) return e;
    if constexpr (sizeof(S) == 2)
      e = seq_tile_rows(p.T, p.B, p.H, D, false) == 128 ? dq<S, D, 2, false>(p, st) : dq<S, D, 1, false>(p, st);
    else
      e = dq<S, D, 1, false>(p, st);
  } else if constexpr (D <= 128) {
    e = dq<S, D, 1, true>(p, st);
  }
  if (e != hipSuccess) return e;
  p.slots = (int)seq_slots(p.T, p.B, 6);
  return p.window ? dkdv<S, D, true>(p, st) : dkdv<S, D, false>(p, st);
}
template <typename S>
static hipError_t bwd_d(const SeqParams& p, int D, hipStream_t st) {
  return D == 32 ? bwd<S, 32>(p, st) : D == 64 ? bwd<S, 64>(p, st) : D == 128 ? bwd<S, 128>(p, st) : bwd<S, 256>(p, st);
}
hipError_t launch_seq_bwd(const SeqParams& p, int dt, int D, hipStream_t st) {
  return dt == DT_BF16 ? bwd_d<bf16>(p, D, st) : dt == DT_F16 ? bwd_d<f16>(p, D, st) : bwd_d<float>(p, D, st);
}

}  // namespace farope
