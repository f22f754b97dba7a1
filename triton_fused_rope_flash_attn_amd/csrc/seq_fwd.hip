// Forward of attention over packed sequences: O and the per-row log-sum-exp.
//
//   s_ij = scale (R q_i).(R k_j), j in i's sequence (causal: j <= i)
//   O_i = sum_j exp(s_ij - m_i) v_j / l_i,   LSE_i = m_i + ln l_i
//
// seq_prep_kernel has written the rotated, scaled K rows; a workgroup of 4 waves
// takes 64 or 128 query rows of one head and streams its sequence's K-hat and V
// rows from memory straight to LDS, in double-buffered stages with one barrier
// each, up to the last row that its queries see.  Short sequences (ROT) have no
// such pass: the workgroups rotate K themselves.
//
// With a window (WIN) a tile reads the stages that hold sinks and those of its rows' windows (KeyStages in seq.h), and a
// row may see no key of its first stages: one of 16384 tokens, 8 heads, D 128, window 1024 113 us, 16 up to 4096,
// 16 heads, D 128, window 512 186 with K-hat's pass.
//
// Bound by the issue of matrix and vector instructions, which overlap between a SIMD's waves:
// one sequence of 16384 tokens, 8 heads, D 128, causal 540 us (1020 TFLOP/s; matrix instructions run
// in 50% of the cycles, vector ones in 41%).  Short sequences wait for latencies: 64 up to 577
// tokens, 12 heads, D 64 25 us (206 TFLOP/s, waves waiting 53% of their time).
#include <type_traits>

#include "seq.h"

namespace farope {

// Keys of a stage: at head_dim 128 in 16 bits 32, which lets three workgroups run on a CU instead
// of two.  Measured (us, forward, 64 / 32 keys): 24 sequences up to 2048 tokens (mean 943), 16 heads 190 / 174,
// 32 up to 512, 16 46 / 40, 8 x 1024, 8 46 / 41, 1 x 4096, 16 101 / 103, 1 x 16384, 8 517 / 527.
template <typename S, int D> constexpr int kFwdRows = sizeof(S) == 2 && D == 128 ? 32 : kStageRowsOf<S, D>;

// O of one row again, key by key and only over the keys that it sees: for the rows of a causal
// call whose sums hold a NaN that may be 0 times an infinity or NaN of a V row behind them.
// A lane takes channel pairs; m and l are the row's reference and sum.  Rarely needed, and slow: one
// infinity behind 9000 of 16384 tokens, 8 heads, D 128 takes the call from 0.55 to 80 ms (32 rows,
// a quarter of a microsecond a key), a channel of NaN throughout to 156.  What
// finds such rows costs (us, without / with) 24 up to 2048 (mean 943), 16 heads, D 128 173 / 175, 64 up to 577, 12
// heads, D 64 40.3 / 40.6, one of 16384, D 128 553 / 549.
template <typename S, int D, bool ROT, bool WIN>
__device__ __forceinline__ void row_again(const SeqParams& p, const SeqTile& tl, int head, int kvh, int i, float m, float l, int lane) {
  constexpr int NP = D > 128 ? D / 128 : 1, AHEAD = 4;
  typedef float f2 __attribute__((ext_vector_type(2)));
  auto turned = [&](const void* base, const int64_t* st, int64_t tok, int h, int index, int c) {
    const S* const x = static_cast<const S*>(base) + tok * st[0] + h * st[1] + c * st[2];
    const float a = (float)x[0], b = (float)x[st[2]];
    const int row = table_row(p.positions ? p.positions[tok] : index - p.has_cls, p.n_pos);
    const int64_t at = (int64_t)row * (D / 2) + c / 2;
    const float co = row < 0 ? 1.f : p.cosp[at], si = row < 0 ? 0.f : p.sinp[at];
    return f2{a * co - b * si, b * co + a * si};
  };
  const bool on = lane < D / 2;
  f2 q[NP], acc[NP];
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    const f2 x = turned(p.q, p.sq, tl.start + i, head, i, on ? 2 * (lane + 64 * n) : 0);
    q[n] = f2{(float)(S)x[0], (float)(S)x[1]};
    acc[n] = f2{0.f, 0.f};
  }
  auto keys = [&](int first, int end) __attribute__((always_inline)) {
    for (int j0 = first; j0 < end; j0 += AHEAD) {
      float s[AHEAD];
      f2 v[AHEAD][NP];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int j = j0 + u < end ? j0 + u : end - 1;
        const int64_t tok = tl.start + j;
        s[u] = 0.f;
#pragma unroll
        for (int n = 0; n < NP; ++n) {
          const int c = on ? 2 * (lane + 64 * n) : 0;
          f2 k;
          if constexpr (ROT) {
            k = turned(p.k, p.sk, tok, kvh, j, c) * p.c2;
            k = f2{(float)(S)k[0], (float)(S)k[1]};
          } else {
            const S* const x = static_cast<const S*>(p.khat) + ((int64_t)kvh * p.T + tok) * D + c;
            k = f2{(float)x[0], (float)x[1]};
          }
          s[u] += on ? q[n][0] * k[0] + q[n][1] * k[1] : 0.f;
          const S* const y = static_cast<const S*>(p.v) + tok * p.sv[0] + kvh * p.sv[1] + c * p.sv[2];
          v[u][n] = f2{(float)y[0], (float)y[p.sv[2]]};
        }
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
#pragma unroll
        for (int d = 1; d < 64; d *= 2) s[u] += __int_as_float(__builtin_amdgcn_ds_bpermute(4 * (lane ^ d), __float_as_int(s[u])));
        const float w = (float)(S)fast_exp2(s[u] - m);
        if (j0 + u < end)
#pragma unroll
          for (int n = 0; n < NP; ++n) acc[n] = f2{acc[n][0] + w * v[u][n][0], acc[n][1] + w * v[u][n][1]};
      }
    }
  };
  const int low = WIN && i + 1 > p.window ? i + 1 - p.window : 0;
  if (WIN) keys(0, p.sinks < low ? p.sinks : low);
  keys(low, i + 1);
  S* const o = static_cast<S*>(p.o) + ((int64_t)(tl.start + i) * p.H + head) * D;
  if (on)
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      o[2 * (lane + 64 * n)] = (S)(acc[n][0] / l);
      o[2 * (lane + 64 * n) + 1] = (S)(acc[n][1] / l);
    }
}

// Wave w owns QT 16-query subtiles.  Logits are computed transposed, S^T = K-hat
// Q-hat^T, so that their output rows (keys) are the k-slots of O^T += V^T P^T and P
// never leaves registers.  The accumulators start at minus the running max, P =
// exp2 of the product's output; O and the row sum are rescaled only when some logit
// exceeds the running max by kSeqSlack.
//
// 16-bit tensors: Q-hat, K-hat and P are rounded once to their type, as the products' operands.
// Together with O's own rounding (1.6e-3 of its norm in bf16) that leaves 2.8e-3.  P as a pair of
// values (hi + lo) measured 2.5e-3, Q-hat too 2.1e-3, at (us, one / P / both) 8 x 1024, 16 heads, D 64
// 40 / 46 / 51, 64 up to 577, 12 heads, D 64 38 / 43 / 46, 16384 tokens, 8 heads, D 128 538 / 700 / 1573.
template <typename S, int D, int QT, bool ROT, bool WIN>
__global__ void __launch_bounds__(kSeqThreads, (sizeof(S) == 4 || D == 256) ? 1 : 3)
seq_fwd_kernel(const SeqParams p) {
  using C = typename SeqComp<S>::C;
  using Frag = typename C::Frag;
  using T = Tile<S, D, kFwdRows<S, D>>;
  constexpr int KS = D / 32, DT = D / 16, SR = T::SR, NB = SR / 32, LB = QT == 2 ? 7 : 6;
  __shared__ __attribute__((aligned(16))) S sK0[SR * D], sK1[SR * D], sV0[SR * D], sV1[SR * D];

  const int tid = thread_id();
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int lr = lane & 15, lg = lane >> 4;
  // heads vary fastest, key heads before the query heads of a group: the workgroups of one
  // key head meet on one XCD when Hkv is a multiple of 8; later rows (more keys) come first
  const int slot = block_id() / p.H, hx = block_id() % p.H;
  const int kvh = hx % p.Hkv, head = kvh * (p.H / p.Hkv) + hx / p.Hkv;
  const SeqTile tl = slot_tile(p, LB, slot, lane, false);
  if (tl.tile < 0) return;
  const int q0 = tl.tile << LB, rows = tl.len - q0 < (1 << LB) ? tl.len - q0 : 1 << LB;
  S* const ob = static_cast<S*>(p.o) + ((int64_t)(tl.start + q0) * p.H + head) * D;
  const unsigned o_row = (unsigned)(p.H * D * (int)sizeof(S));
  const auto rO = make_rsrc(ob, (unsigned)(rows - 1) * o_row + T::RB);
  const auto rL = make_rsrc(p.lse + (int64_t)head * p.T + tl.start + q0, (unsigned)rows * 4u);
  const int row0 = wave * 16 * QT + lr;   // of the tile; subtile t: + 16 t

  if (tl.seq == p.B) {   // tokens behind the last sequence: zeros
    for (int r = tid / (D / 8); r < rows; r += kSeqThreads / (D / 8)) {
      const float z[8] = {};
      put_row8<S>(ob + (int64_t)r * p.H * D + 8 * (tid % (D / 8)), z);
    }
    if (tid < rows) p.lse[(int64_t)head * p.T + tl.start + q0 + tid] = 0.f;
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

  Frag qf[QT][KS];
  int seen[QT];   // keys that the subtile's row of this lane sees
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int i = q0 + row0 + 16 * t, ic = i < tl.len ? i : tl.len - 1, tok = tl.start + ic;
    seen[t] = p.causal ? ic + 1 : tl.len;
    const S* qp = static_cast<const S*>(p.q) + tok * p.sq[0] + head * p.sq[1];
    const int tr = table_row(p.positions ? p.positions[tok] : ic - p.has_cls, p.n_pos);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float x[8], cs[8];
      load8<S>(qp + (32 * s + 8 * lg) * p.sq[2], p.sq[2], p.vec_q, x);
      table_load4(p.cosp, p.sinp, tr, D / 2, 16 * s + 4 * lg, cs);
      rope_rotate8(x, cs);
      qf[t][s] = C::make(x);
    }
  }
  const int w0 = q0 + wave * 16 * QT;   // the wave's first row (uniform)
  const bool active = w0 < tl.len;
  // every row of the wave sees keys below lo, none sees keys from hi on
  const int lo = p.causal ? w0 + 1 : tl.len;
  const int hi = p.causal && w0 + 16 * QT < tl.len ? w0 + 16 * QT : tl.len;
  const int ns = ks.n;

  f32x4 acc[QT][DT];
  float m_run[QT], l_run[QT];   // the running max (less kWeightUp) and sum
  f32x4 nm4[QT];       // minus the running max (0 before the first block)
  float thr = -INFINITY;   // a value above it makes the block rescale
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    m_run[t] = -INFINITY;
    l_run[t] = 0.f;
    nm4[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  FragAt<S, D> at;
  at.init(lr, lg);

  // One stage's keys: the logit products, one test of the running max, then the
  // probabilities and O products of its 32-key blocks.
  auto blocks = [&](bool tail, bool edge, int k0, const S* __restrict__ k, const S* __restrict__ v) __attribute__((always_inline)) {
    f32x4 sacc[NB][QT][2];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const Frag a = at.row(k + 32 * j * D, s, h);
#pragma unroll
          for (int t = 0; t < QT; ++t) sacc[j][t][h] = C::mma(a, qf[t][s], s == 0 ? nm4[t] : sacc[j][t][h]);
        }
    if (tail) {   // uniform: some of these keys are behind a row of the wave
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const int lim = seen[t] - k0 - 4 * lg;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) sacc[j][t][h][i] = 32 * j + 16 * h + i < lim ? sacc[j][t][h][i] : -INFINITY;
      }
    }
    if (WIN && edge) {   // uniform: some are before a row's window
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const int from = seen[t] - p.window - k0 - 4 * lg, sinks = p.sinks - k0 - 4 * lg;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int e = 32 * j + 16 * h + i;
              sacc[j][t][h][i] = e >= from || e < sinks ? sacc[j][t][h][i] : -INFINITY;
            }
      }
    }
    float mx[QT], mxx = -INFINITY;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      mx[t] = -INFINITY;
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x4 x = sacc[j][t][h];
          mx[t] = fmaxf(mx[t], fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
        }
      mxx = fmaxf(mxx, mx[t]);
    }
    if (__any(mxx > thr)) {
      thr = kSeqSlack + kWeightUp<S>;
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const float old = m_run[t] == -INFINITY ? 0.f : m_run[t];
        const float mnew = fmaxf(m_run[t], group4_max(mx[t]) + old - kWeightUp<S>);
        const bool none = WIN && mnew == -INFINITY;   // the row has seen nothing yet: its first key is to rescale
        const float alpha = none ? 1.f : fast_exp2(m_run[t] - mnew), sh = none ? 0.f : old - mnew, nm = none ? 0.f : -mnew;
        if (none) thr = -INFINITY;
        m_run[t] = mnew;
        l_run[t] *= alpha;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[t][d] *= alpha;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) sacc[j][t][h] += sh;
        nm4[t] = f32x4{nm, nm, nm, nm};
      }
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      Frag pf[QT];
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        float x[8];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[4 * h + i] = fast_exp2(sacc[j][t][h][i]);
        l_run[t] += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        pf[t] = C::make(x);   // (16-bit tensors: P rounded to their type for the O product; the row sum is not)
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const Frag a = at.col(v + 32 * j * D, d);
#pragma unroll
        for (int t = 0; t < QT; ++t) acc[t][d] = C::mma(a, pf[t], acc[t][d]);
      }
    }
  };
  auto stage = [&](int st, const S* __restrict__ k, const S* __restrict__ v, S* __restrict__ kn, S* __restrict__ vn)
      __attribute__((always_inline)) {
    seq_stage_barrier();
    if (st + 1 < ns) {
      if constexpr (ROT) rot.load(p, tl, kvh, ks.at(st + 1), tid);
      else srcK.load(kn, wave, ks.at(st + 1) * SR);
      srcV.load(vn, wave, ks.at(st + 1) * SR);
    }
    const int k0 = ks.at(st) * SR;
    if constexpr (WIN) {   // (keys before all windows of the wave's rows, and some that are before one's)
      const bool seen_by_some = k0 < hi && (k0 + SR > w0 + 1 - p.window || k0 < p.sinks);
      if (active && seen_by_some) blocks(k0 + SR > lo, past_window(p, k0, SR, hi - p.window), k0, k, v);
    } else {
      if (active && k0 < hi) blocks(k0 + SR > lo, false, k0, k, v);
    }
    if (ROT && st + 1 < ns) rot.store(p, kn, tid);   // (read in the stage before this one)
  };
  if constexpr (ROT) rot.store(p, sK0, tid);
  for (int st = 0; st < ns; st += 2) {
    stage(st, sK0, sV0, sK1, sV1);
    if (st + 1 < ns) stage(st + 1, sK1, sV1, sK0, sV0);
  }

  // lane holds O[row][16d + 4lg + (0..3)]; rows past the tile drop
  unsigned again[QT];   // rows (bits) of the subtile that row_again takes
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int row = row0 + 16 * t;
    const float l = group4_sum(l_run[t]);
    again[t] = 0;
    if (p.causal) {   // (a sum is not finite if a term is not)
      f32x4 x = acc[t][0];
#pragma unroll
      for (int d = 1; d < DT; ++d) x += acc[t][d];
      const float sum = (x[0] + x[1]) + (x[2] + x[3]);
      const uint64_t bad =
          __builtin_amdgcn_ballot_w64(magnitude_bits(sum) >= kInfBits && magnitude_bits(l) - 1u < kInfBits - 1u && row < rows);
      again[t] = (unsigned)(bad | bad >> 16 | bad >> 32 | bad >> 48) & 0xffffu;
    }
    const float inv = __builtin_amdgcn_rcpf(l);
    if constexpr (sizeof(S) == 4) {
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const f32x4 x = acc[t][d] * inv;
        buf_store16(__builtin_bit_cast(u32x4, x), rO, (unsigned)row * o_row + (unsigned)(16 * d + 4 * lg) * 4u, 0u);
      }
    } else {
      // lane groups lg and lg^1 trade halves so that each lane stores 8 consecutive channels
#pragma unroll
      for (int d0 = 0; d0 < DT; d0 += 2) {
        u32x2 w[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          typedef S s4 __attribute__((ext_vector_type(4)));
          s4 a;
#pragma unroll
          for (int r = 0; r < 4; ++r) a[r] = (S)(acc[t][d0 + j][r] * inv);
          __builtin_memcpy(&w[j], &a, 8);
        }
        u32x4 x;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const auto r = __builtin_amdgcn_permlane16_swap(w[0][k], w[1][k], false, false);
          x[k] = r[0];
          x[2 + k] = r[1];
        }
        buf_store16(x, rO, (unsigned)row * o_row + (unsigned)(16 * (d0 + (lg & 1)) + 4 * (lg & 2)) * 2u, 0u);
      }
    }
    // (lanes lg != 0 write past the range)
    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint((m_run[t] + fast_log2(l)) * kLn2), rL,
                                          (unsigned)(lg == 0 ? row : 1 << LB) * 4u, 0u, 0);
  }
  unsigned any = 0;
#pragma unroll
  for (int t = 0; t < QT; ++t) any |= again[t];
  if (any == 0) return;   // (uniform)
  // Some key that a row of the wave has met without seeing it holds one.  (Where the key that
  // all of them see is NaN throughout, so is O, and rightly.)
  auto v_bits = [&](int j, int c) {
    return magnitude_bits((float)static_cast<const S*>(p.v)[(tl.start + j) * p.sv[0] + kvh * p.sv[1] + c * p.sv[2]]);
  };
  bool odd = false, some = WIN;
  for (int c = lane; c < D; c += 64) {
    if constexpr (WIN) {
      for (int st = 0; st < ns; ++st)
        for (int j = ks.at(st) * SR; j < ks.at(st) * SR + SR && j < tl.len; ++j) odd |= v_bits(j, c) >= kInfBits;
    } else {
      some |= v_bits(w0, c) <= kInfBits;
      for (int j = w0 + 1; j < ns * SR && j < tl.len; ++j) odd |= v_bits(j, c) >= kInfBits;
    }
  }
  if (!__any(odd) || !__any(some)) return;
  __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): the rows as stored above come first
  asm volatile("" : : : "memory");
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const float l = group4_sum(l_run[t]);
    for (unsigned left = again[t]; left; left &= left - 1) {
      const int r = __builtin_ctz(left);
      row_again<S, D, ROT, WIN>(p, tl, head, kvh, w0 + 16 * t + r, __int_as_float(__builtin_amdgcn_readlane(__float_as_int(m_run[t]), r)),
                           __int_as_float(__builtin_amdgcn_readlane(__float_as_int(l), r)), lane);
    }
  }
}

template <typename S, int D, int QT, bool ROT>
static hipError_t fwd(const SeqParams& p0, hipStream_t st) {
  SeqParams p = p0;
  p.slots = (int)seq_slots(p.T, p.B, QT == 2 ? 7 : 6);
  const dim3 grid((unsigned)p.slots * p.H);
  if (p.window) hipLaunchKernelGGL((seq_fwd_kernel<S, D, QT, ROT, true>), grid, dim3(kSeqThreads), 0, st, p);
  else hipLaunchKernelGGL((seq_fwd_kernel<S, D, QT, ROT, false>), grid, dim3(kSeqThreads), 0, st, p);
  return hipGetLastError();
}
template <typename S, int D>
static hipError_t fwd_rows(const SeqParams& p, hipStream_t st) {
  if constexpr (D <= 128)
    if (!p.khat) return fwd<S, D, 1, true>(p, st);
  if constexpr (sizeof(S) == 2)
    if (seq_tile_rows(p.T, p.B, p.H, D, false) == 128) return fwd<S, D, 2, false>(p, st);
  return fwd<S, D, 1, false>(p, st);
}
template <typename S>
static hipError_t fwd_d(const SeqParams& p, int D, hipStream_t st) {
  return D == 32 ? fwd_rows<S, 32>(p, st) : D == 64 ? fwd_rows<S, 64>(p, st)
         : D == 128 ? fwd_rows<S, 128>(p, st) : fwd_rows<S, 256>(p, st);
}
hipError_t launch_seq_fwd(const SeqParams& p, int dt, int D, hipStream_t st) {
  return dt == DT_BF16 ? fwd_d<bf16>(p, D, st) : dt == DT_F16 ? fwd_d<f16>(p, D, st) : fwd_d<float>(p, D, st);
}

}  // namespace farope
