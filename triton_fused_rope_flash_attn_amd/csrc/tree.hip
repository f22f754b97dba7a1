// Attention of several new tokens per sequence over its paged cache: a tree of
// drafted tokens, or a chain of them (a prompt in chunks).
//
//   q-hat = R(position) q;  O_j = softmax(scale q-hat_j K^T) V over the rows that token j of its sequence sees: the
//   `lengths` cached before the new tokens, and of the new ones' rows, which lie behind them, those that
//   tree[j] names (chain: rows 0 .. j).  K is cached rotated.  A token that sees no row has O = 0.
//
// A key head's query rows (tokens times the heads of its group, head fastest) are taken in tiles of
// 64 or 128, whose 4 waves have 16 or 32 of them each, and the cache's rows in stages, gathered through the page
// table from memory straight to LDS, three stages ahead, one barrier a stage.  The stages of all tiles of all
// sequences are divided evenly over the workers (workgroups) of a key head, as in decode.hip: a
// worker's share may end inside a tile and run on in the next; of tiles that several workers share
// these leave unnormalised sums, which tree_join_kernel joins.
//
// Few rows are bound by memory (the cache is read once a tile), many by the issue of matrix and vector
// instructions and by the last-level cache, from which every tile has its rows.  Measured (us a call, both launches): 32
// sequences up to 8192 rows with up to 32 drafted tokens, 32 heads of 8, D 128, bf16 150 (497 MB; without the
// products 122); 4 up to 8192 with up to 1024 new tokens, fp16 330 (670 TFLOP/s; without 205); one of 1024
// with 8, 12 heads, D 64 14.6, the chain of lengths, page numbers, rows and the join.
//
// 16-bit tensors: q-hat (with the scale) and P are rounded once to their type, as the products' operands, as in the forward over
// packed sequences; with O's own rounding that leaves 2.8e-3 of O's norm in bf16 (the storing alone 1.7e-3).  As pairs of values, as
// in decode.hip, where a step has 16 rows a key head: P alone 2.4e-3, q-hat alone 2.2e-3, both 1.7e-3; us, one / P / q-hat / both: the
// three calls above 150 / 156 / 156 / 163, 325 / 439 / 388 / 497, 14.7 / 14.8 / 14.8 / 15.0; 32 of 8192 with 32 new tokens 243 / both 322, 32 of
// 4096 with 16, D 64 64 / 70 / 68 / 75, 8 of 4096 with 32, 16 heads of 4, D 256 93 / 101 / 149 / 155.
#include <type_traits>

#include "seq.h"

namespace farope {

// Rows of a stage and stages in LDS: three are on their way while one is read, but for rows of 1 KB.  (One stage of 64 rows
// on its way: 152 us and 337 for the first two calls above; two stages and three workgroups a CU 158 and 340.)
template <typename S, int D> constexpr int kTreeRows = D * sizeof(S) <= 128 ? 64 : 32;
template <typename S, int D> constexpr int kTreeBufs = D * sizeof(S) <= 512 ? 4 : 2;

// What a sequence has: its tokens, rows cached before them, rows in the cache with them, tiles, stages of a tile.
struct TreeSeq {
  int start, m, len, n, tiles, blocks;
};
template <int ROWS, int SR>
__device__ __forceinline__ TreeSeq tree_seq(const TreeParams& p, int b) {
  TreeSeq s;
  s.start = cu_at(p.cu, b, p.T);
  const int end = cu_at(p.cu, b + 1, p.T);
  s.m = end > s.start ? end - s.start : 0;
  s.len = p.c.lengths[b];
  const int64_t room = (int64_t)p.c.max_pages * p.c.page, all = (int64_t)s.len + s.m;
  const int64_t n = s.len < 0 ? 0 : all < room ? all : room;
  s.n = n < INT32_MAX - 255 ? (int)n : INT32_MAX - 255;   // (so that a stage's last row has a number)
  s.tiles = (int)(((int64_t)s.m * (p.H / p.Hkv) + ROWS - 1) / ROWS);
  s.blocks = s.n > 0 ? (s.n + SR - 1) / SR : 1;   // (a tile without rows is visited too, for its zeros)
  return s;
}

__device__ __forceinline__ TreeSeq uniform(TreeSeq s) {
  s.start = __builtin_amdgcn_readfirstlane(s.start);
  s.m = __builtin_amdgcn_readfirstlane(s.m);
  s.len = __builtin_amdgcn_readfirstlane(s.len);
  s.n = __builtin_amdgcn_readfirstlane(s.n);
  s.tiles = __builtin_amdgcn_readfirstlane(s.tiles);
  s.blocks = __builtin_amdgcn_readfirstlane(s.blocks);
  return s;
}

__device__ __forceinline__ int64_t wave_scan64(int64_t x, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int64_t y = shfl64(x, lane - d);
    if (lane >= d) x += y;
  }
  return x;
}
__device__ __forceinline__ int64_t lane64(int64_t x, int l) {
  return (int64_t)((uint64_t)(unsigned)__builtin_amdgcn_readlane((int)(x >> 32), l) << 32 | (unsigned)__builtin_amdgcn_readlane((int)x, l));
}

// The tile of a slot: sequence i takes slots (cu[i] * group >> lb) + i on, as in find_tile (seq.h).
__device__ __forceinline__ void find_rows(const TreeParams& p, int lb, int slot, int lane, int& seq, int& tile) {
  const int group = p.H / p.Hkv;
  int lo = 0, n = p.B + 1;
  while (n > 1) {
    const int step = (n + 63) >> 6, j = lane * step;
    const bool le = j < n && ((cu_at(p.cu, lo + (j < n ? j : 0), p.T) * group) >> lb) + lo + j <= slot;
    const int k = 63 - __builtin_clzll(__builtin_amdgcn_ballot_w64(le) | 1ull);
    lo += k * step;
    n = n - k * step < step ? n - k * step : step;
  }
  seq = __builtin_amdgcn_readfirstlane(lo);
  tile = slot - (((cu_at(p.cu, seq, p.T) * group) >> lb) + seq);
}

__device__ const float kZeros[4] __attribute__((aligned(16))) = {0.f, 0.f, 0.f, 0.f};

// One byte of a buffer (a plain function, as lds_dma16).
__device__ __forceinline__ uint8_t buf_load1(__amdgpu_buffer_rsrc_t r, unsigned voff) {
  return __builtin_amdgcn_raw_buffer_load_b8(r, voff, 0, 0);
}

// Every wave is here, with at most N of its loads still on their way and none of its LDS accesses.  (Without the
// fences of lds_barrier, which wait for all loads to LDS.)
template <int N> __device__ __forceinline__ void loads_barrier() {
  static_assert(N < 64, "");
  asm volatile("" : : : "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);
  __builtin_amdgcn_s_barrier();
  asm volatile("" : : : "memory");
}

__device__ __forceinline__ int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// 16 bytes per lane from memory straight into LDS (lane l lands at lds + 16 l).
__device__ __forceinline__ void gather16(const void* from, void* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) unsigned*)from,
                                   (__attribute__((address_space(3))) unsigned*)lds, 16, 0, 0);
}

// O (or the sums) of one row of a tile again, row by row of the cache and only over those that it sees: for
// rows whose sums hold an infinity or a NaN, which may be 0 times a value of a row that they do not see, or of one
// that they see with a weight that rounds to 0.  m: the row's reference; out: `factor` times the sums,
// rounded where they are O.  A lane takes channel pairs.  Rarely needed, and slow.
template <typename S, int D>
__device__ __forceinline__ void tree_row_again(const TreeParams& p, const TreeSeq& s, int b, int kvh, int head, int j, int seen,
                                               int from, int to, float m, float factor, void* out, bool is_o, int lane) {
  constexpr int NP = D > 128 ? D / 128 : 1;
  typedef float f2 __attribute__((ext_vector_type(2)));
  const bool on = lane < D / 2;
  const int64_t tok = s.start + j, index = (int64_t)s.len + j - p.has_cls;
  const int tr = table_row(p.positions ? p.positions[tok] : (int)(index < INT32_MAX ? index : INT32_MAX), p.n_pos);
  f2 q[NP], acc[NP];
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    const int c = on ? 2 * (lane + 64 * n) : 0;
    const S* const x = static_cast<const S*>(p.q) + tok * p.sq[0] + head * p.sq[1] + c * p.sq[2];
    const float x0 = (float)x[0], x1 = (float)x[p.sq[2]];
    const int64_t at = (int64_t)tr * (D / 2) + c / 2;
    const float co = tr < 0 ? 1.f : p.cosp[at], si = tr < 0 ? 0.f : p.sinp[at];
    q[n] = f2{(float)(S)((x0 * co - x1 * si) * p.c2), (float)(S)((x1 * co + x0 * si) * p.c2)};
    acc[n] = f2{0.f, 0.f};
  }
  for (int r = from; r < to; ++r) {
    if (p.tree ? r >= s.len && (r - s.len >= p.cols || !p.tree[tok * p.stree + r - s.len]) : r >= seen) continue;
    const int place = r / p.c.page, g = p.c.pages[b * p.c.spages + place];
    if (g < 0 || g >= p.c.n_pages) continue;
    const int64_t in = r - (int64_t)place * p.c.page;
    const S* const k = static_cast<const S*>(p.c.kc) + g * p.c.skc[0] + in * p.c.skc[1] + kvh * p.c.skc[2];
    const S* const v = static_cast<const S*>(p.c.vc) + g * p.c.svc[0] + in * p.c.svc[1] + kvh * p.c.svc[2];
    float x = 0.f;
    f2 y[NP];
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      const int c = on ? 2 * (lane + 64 * n) : 0;
      x += on ? q[n][0] * (float)k[c] + q[n][1] * (float)k[c + 1] : 0.f;
      y[n] = f2{(float)v[c], (float)v[c + 1]};
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) x += __int_as_float(__builtin_amdgcn_ds_bpermute(4 * (lane ^ d), __float_as_int(x)));
    const float w = (float)(S)fast_exp2(x - m);
#pragma unroll
    for (int n = 0; n < NP; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) acc[n][e] += (magnitude_bits(y[n][e]) >= kInfBits ? fmaxf(w, 0x1p-126f) : w) * y[n][e];
  }
#pragma unroll
  for (int n = 0; n < NP; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int c = 2 * (lane + 64 * n) + e;
      const float x = acc[n][e] * factor;
      if (!on) continue;
      if (is_o) static_cast<S*>(out)[c] = (S)x;
      else static_cast<float*>(out)[c] = x;
    }
}

template <typename S, int D, int QT>
__global__ void __launch_bounds__(kSeqThreads, D * sizeof(S) <= 256 ? 2 : 1) tree_kernel(const TreeParams p) {
  using C = typename SeqComp<S>::C;
  using Frag = typename C::Frag;
  using T = Tile<S, D, kTreeRows<S, D>>;
  constexpr int BUFS = kTreeBufs<S, D>, AHEAD = BUFS - 1, LOADS = 2 * T::NI;   // (LOADS: of a wave and stage)
  constexpr int KS = D / 32, DT = D / 16, SR = T::SR, NB = SR / 32, ROWS = 64 * QT, LB = QT == 2 ? 7 : 6;
  constexpr uint64_t kAll = SR == 64 ? ~0ull : 0xffffffffull;
  constexpr int MORE = BUFS > 2 ? SR * D : 8;
  __shared__ __attribute__((aligned(16))) S sK0[SR * D], sK1[SR * D], sK2[MORE], sK3[MORE];
  __shared__ __attribute__((aligned(16))) S sV0[SR * D], sV1[SR * D], sV2[MORE], sV3[MORE];

  const int tid = thread_id();
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int worker = block_id() / p.Hkv, kvh = block_id() % p.Hkv, group = p.H / p.Hkv;

  // this worker's stages [at, stop) of all, from stage `first` of tile `tile` of sequence b on; `before`: the
  // stages of the tiles before that one
  int b = 0, tile = 0, first = 0, which = 0;
  int64_t at = 0, stop = 0, before = 0, size = 1;
  if (p.direct) {
    find_rows(p, LB, worker, lane, b, tile);
    if (b == p.B) {   // tokens behind the last sequence: zeros
      const int start = cu_at(p.cu, b, p.T), rows = (p.T - start) * group, r0 = tile * ROWS;
      for (int r = r0 + tid / (D / 8); r < rows && r < r0 + ROWS; r += kSeqThreads / (D / 8)) {
        const float z[8] = {};
        put_row8<S>(static_cast<S*>(p.o) + ((int64_t)(start + r / group) * p.H + kvh * group + r % group) * D + 8 * (tid % (D / 8)), z);
      }
      return;
    }
    const TreeSeq s = tree_seq<ROWS, SR>(p, b);
    if (tile >= s.tiles) return;
  } else {
    int64_t all = 0, n = 0, sum = 0;
    for (int i = 0; i < p.B; i += 64) {
      n = 0;
      if (i + lane < p.B) {
        const TreeSeq s = tree_seq<ROWS, SR>(p, i + lane);
        n = (int64_t)s.tiles * s.blocks;
      }
      sum = wave_scan64(n, lane);
      all += lane64(sum, 63);
    }
    const int64_t even = lane64((all + p.workers - 1) / p.workers, 0);
    size = even > kTreeLeast ? even : kTreeLeast;
    at = worker * size;
    if (at >= all) return;
    stop = at + size < all ? at + size : all;
    b = -1;
    for (int i = 0; i < p.B; i += 64) {   // (some sequence holds stage `at`)
      if (p.B > 64) {
        n = 0;
        if (i + lane < p.B) {
          const TreeSeq s = tree_seq<ROWS, SR>(p, i + lane);
          n = (int64_t)s.tiles * s.blocks;
        }
        sum = wave_scan64(n, lane);
      }
      const uint64_t past = __builtin_amdgcn_ballot_w64(before + sum > at);
      if (past) {
        const int l = __builtin_ctzll(past);
        b = i + l;
        before += lane64(sum, l) - lane64(n, l);
        break;
      }
      before += lane64(sum, 63);
    }
    if (b < 0) return;
    const TreeSeq s = uniform(tree_seq<ROWS, SR>(p, b));
    tile = __builtin_amdgcn_readfirstlane((int)((at - before) / s.blocks));
    before += (int64_t)tile * s.blocks;
    first = (int)(at - before);
  }

  for (;;) {
    // (a lane number that the compiler takes as new for each piece: what follows from it, computed once for all of
    // them, filled the registers)
    const int lane = fresh(tid & 63), lr = lane & 15, lg = lane >> 4;
    FragAt<S, D> frag;
    frag.init(lr, lg);
    const TreeSeq s = uniform(tree_seq<ROWS, SR>(p, b));
    const int stages = p.direct || stop - at > s.blocks - first ? s.blocks : first + (int)(stop - at);   // this piece: [first, stages)
    const int r0 = tile * ROWS, rows = s.m * group - r0 < ROWS ? s.m * group - r0 : ROWS;
    const bool chain = !p.tree;
    // rows of the cache that the tile's last token sees (a tree's: all); stages behind them hold nothing for it
    auto seen_by = [&](int row) {   // (int64: a length may be any number)
      const int64_t x = chain ? (int64_t)s.len + (r0 + row) / group + 1 : s.n;
      return x < s.n ? (int)x : s.n;
    };
    const int last = (__builtin_amdgcn_readfirstlane(seen_by(rows - 1)) + SR - 1) / SR, end = stages < last ? stages : last;

    // lane l: row l of a stage: page and row in it
    const int* const pages = p.c.pages + b * p.c.spages;
    struct Ids { int page, row; };   // (row -1: there is none)
    auto fetch = [&](int st) __attribute__((always_inline)) {
      const unsigned r = (unsigned)st * SR + (unsigned)lane;   // (below 2^31: stages end at s.n, with a few behind)
      unsigned place = (unsigned)((uint64_t)r * p.page_mul >> p.page_shift);   // r / page
      Ids id;
      id.row = st < end && lane < SR && r < (unsigned)s.n ? (int)(r - place * (unsigned)p.c.page) : -1;
      place = place < (unsigned)p.c.max_pages ? place : (unsigned)p.c.max_pages - 1u;
      id.page = pages[place];   // (one load whatever there is, so that the number of loads on their way is known)
      return id;
    };
    auto load = [&](Ids id, S* __restrict__ kd, S* __restrict__ vd) __attribute__((always_inline)) {
      id.page = fresh(id.page);   // (not looked at before the barrier, where other loads would have to be waited for)
      const bool in = id.row >= 0 && id.page >= 0 && id.page < p.c.n_pages;
      const uint64_t rows_in = __builtin_amdgcn_ballot_w64(in);
      // (strides in 16 bytes; K rows that do not exist: page 0's first; they are masked)
      const unsigned g = in ? (unsigned)id.page : 0u, r = in ? (unsigned)id.row : 0u;
      const int64_t ko = (int64_t)((uint64_t)g * p.k16[0] + (uint64_t)r * p.k16[1]);
      const int64_t vo = (int64_t)((uint64_t)g * p.v16[0] + (uint64_t)r * p.v16[1]);
      const char* const kb = static_cast<const char*>(p.c.kc) + kvh * p.c.skc[2] * (int)sizeof(S);
      const char* const vb = static_cast<const char*>(p.c.vc) + kvh * p.c.svc[2] * (int)sizeof(S);
      const unsigned ln = (unsigned)fresh(lane) & 63u;
      int64_t kr[T::NI], vr[T::NI];
#pragma unroll
      for (int i = 0; i < T::NI; ++i) vr[i] = kr[i] = shfl64(ko, (i * kSeqNW + wave) * T::RPI + (int)(ln / T::CPR));
      if (!p.alike) {   // (uniform)
#pragma unroll
        for (int i = 0; i < T::NI; ++i) vr[i] = shfl64(vo, (i * kSeqNW + wave) * T::RPI + (int)(ln / T::CPR));
      }
#pragma unroll
      for (int i = 0; i < T::NI; ++i) {
        const int rw = (i * kSeqNW + wave) * T::RPI + (int)(ln / T::CPR), ch = (int)(ln % T::CPR) ^ T::chunk_xor(rw);
        gather16(kb + 16 * (kr[i] + ch), kd + (i * kSeqNW + wave) * T::RPI * D);
        const char* const from = vb + 16 * (vr[i] + ch);   // V rows that do not exist are zeros: their weights are
        gather16(rows_in >> rw & 1 ? from : reinterpret_cast<const char*>(kZeros), vd + (i * kSeqNW + wave) * T::RPI * D);
      }
      return rows_in;   // the stage's rows (bits) that exist
    };

    const auto rTree = make_rsrc(p.tree + (chain ? 0 : s.start * p.stree), chain ? 0u : (unsigned)((s.m - 1) * (int)p.stree + p.cols));
    const int row0 = wave * 16 * QT + lr;   // of the tile; subtile t: + 16 t
    const int w0 = wave * 16 * QT, w1 = w0 + 16 * QT < rows ? w0 + 16 * QT - 1 : rows - 1;
    const bool active = w0 < rows;
    // every row of the wave sees rows below lo of the cache, none sees rows from hi on
    const int lo = chain ? __builtin_amdgcn_readfirstlane(seen_by(active ? w0 : 0)) : s.len < s.n ? s.len : s.n;
    const int hi = __builtin_amdgcn_readfirstlane(seen_by(active ? w1 : 0));
    Frag qf[QT][KS];
    int seen[QT];                // chain: rows that the lane's row of the subtile sees
    int tok[QT];                 // its token of the sequence
    f32x4 acc[QT][DT];
    float m_run[QT], l_run[QT];
    {
      // ids[i] and rows_in[i]: of the stages that are first + i but for a multiple of 4.  Page numbers are read AHEAD
      // stages before their rows, so that to wait for them is not to wait for rows.  Stages behind the piece's
      // end are loaded too (V as zeros, K from one row), and not used.
      Ids ids[4];
      uint64_t rows_in[4];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) ids[i] = fetch(first + i);
      rows_in[0] = load(ids[0], sK0, sV0);
      if constexpr (AHEAD > 1) {   // (one stage's loads after the other's: the waits count on it)
        asm volatile("" : : : "memory");
        rows_in[1] = load(ids[1], sK1, sV1);
        asm volatile("" : : : "memory");
        rows_in[2] = load(ids[2], sK2, sV2);
      }
#pragma unroll
      for (int i = AHEAD; i < 2 * AHEAD; ++i) ids[i & 3] = fetch(first + i);
      {
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          const int r = row0 + 16 * t < rows ? row0 + 16 * t : rows - 1, j = (r0 + r) / group, h = kvh * group + (r0 + r) % group;
          const int64_t at_tok = s.start + j, index = (int64_t)s.len + j - p.has_cls;
          seen[t] = seen_by(r);
          tok[t] = j;
          const int tr = table_row(p.positions ? p.positions[at_tok] : (int)(index < INT32_MAX ? index : INT32_MAX), p.n_pos);
          const S* const qp = static_cast<const S*>(p.q) + at_tok * p.sq[0] + h * p.sq[1];
#pragma unroll
          for (int c = 0; c < KS; ++c) {
            float x[8], cs[8];
            load8<S>(qp + (32 * c + 8 * lg) * p.sq[2], p.sq[2], p.vec_q, x);
            table_load4(p.cosp, p.sinp, tr, D / 2, 16 * c + 4 * lg, cs);
            rope_rotate8(x, cs);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= p.c2;
            qf[t][c] = C::make(x);   // (16-bit tensors: rounded once, with the scale)
          }
        }
      }
      float thr = -INFINITY;   // a value above it makes the stage rescale
      f32x4 nm4[QT];
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        m_run[t] = -INFINITY;
        l_run[t] = 0.f;
        nm4[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
      }

      auto blocks = [&](bool tail, uint64_t have, int k0, const S* __restrict__ k, const S* __restrict__ v) __attribute__((always_inline)) {
        f32x4 sacc[NB][QT][2];
#pragma unroll
        for (int c = 0; c < KS; ++c)
#pragma unroll
          for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const Frag a = frag.row(k + 32 * j * D, c, h);
#pragma unroll
              for (int t = 0; t < QT; ++t) sacc[j][t][h] = C::mma(a, qf[t][c], c == 0 ? nm4[t] : sacc[j][t][h]);
            }
        if (tail) {   // uniform: some row of the wave does not see all of these rows
#pragma unroll
          for (int t = 0; t < QT; ++t) {
            const int g4 = fresh(4 * lg), lim = (chain ? seen[t] : s.len) - k0 - g4;
            unsigned more = 0;   // bit 8 j + 4 h + i: the lane's row sees row 32 j + 16 h + 4 lg + i of the stage, a new token's
            if (!chain && k0 + SR > s.len && p.cols > 0) {   // (uniform) the bytes of its row of the tree, all loads in flight together
              const int d0 = -lim;
              const int at_row = tok[t] * (int)p.stree;
              uint8_t x[8 * NB];
#pragma unroll
              for (int e = 0; e < 8 * NB; ++e) {   // (what lies behind the sequence's rows reads as 0)
                const int d = d0 + 32 * (e >> 3) + 16 * (e >> 2 & 1) + (e & 3);
                x[e] = buf_load1(rTree, (unsigned)(at_row + (d > 0 ? d : 0)));
              }
#pragma unroll
              for (int e = 0; e < 8 * NB; ++e) {
                const int d = d0 + 32 * (e >> 3) + 16 * (e >> 2 & 1) + (e & 3);
                more |= d >= 0 && d < p.cols && x[e] != 0 ? 1u << e : 0u;
              }
            }
            const uint64_t there = have >> g4;
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const int e = 32 * j + 16 * h + i;
                  const bool in = (e < lim || (more >> (8 * j + 4 * h + i) & 1)) && (there >> e & 1);
                  sacc[j][t][h][i] = in ? sacc[j][t][h][i] : -INFINITY;
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
        if (__any(mxx > thr)) {   // (as in the forward over packed sequences)
          thr = kSeqSlack + kWeightUp<S>;
#pragma unroll
          for (int t = 0; t < QT; ++t) {
            const float old = m_run[t] == -INFINITY ? 0.f : m_run[t];
            const float mnew = fmaxf(m_run[t], group4_max(mx[t]) + old - kWeightUp<S>);
            const bool none = mnew == -INFINITY;   // the row has seen nothing yet
            const float alpha = none ? 1.f : fast_exp2(m_run[t] - mnew), sh = none ? 0.f : old - mnew, nm = none ? 0.f : -mnew;
            m_run[t] = mnew;
            thr = none ? -INFINITY : thr;
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
          Frag a[3];   // (two fragments ahead)
          a[0] = frag.col(v + 32 * j * D, 0);
          a[1] = frag.col(v + 32 * j * D, 1);
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            if (d + 2 < DT) a[(d + 2) % 3] = frag.col(v + 32 * j * D, d + 2);
#pragma unroll
            for (int t = 0; t < QT; ++t) acc[t][d] = C::mma(a[d % 3], pf[t], acc[t][d]);
          }
        }
      };
      auto stage = [&](auto slot, int st, const S* __restrict__ k, const S* __restrict__ v, S* __restrict__ kn, S* __restrict__ vn)
          __attribute__((always_inline)) {
        constexpr int U = decltype(slot)::value;
        // The stage's own loads have landed: those of the AHEAD - 1 stages behind it are the last that were issued, LOADS
        // each at least (page numbers come on top).
        loads_barrier<(AHEAD - 1) * LOADS>();
        const uint64_t have = rows_in[U];
        rows_in[(U + AHEAD) & 3] = load(ids[(U + AHEAD) & 3], kn, vn);
        ids[(U + 2 * AHEAD) & 3] = fetch(st + 2 * AHEAD);
        const int k0 = st * SR;
        if (active && st < end && k0 < hi) blocks(have != kAll || k0 + SR > lo, have, k0, k, v);
      };
      using std::integral_constant;
      for (int st = first; st < end; st += 4) {
        if constexpr (BUFS == 4) {
          stage(integral_constant<int, 0>{}, st, sK0, sV0, sK3, sV3);
          stage(integral_constant<int, 1>{}, st + 1, sK1, sV1, sK0, sV0);
          stage(integral_constant<int, 2>{}, st + 2, sK2, sV2, sK1, sV1);
          stage(integral_constant<int, 3>{}, st + 3, sK3, sV3, sK2, sV2);
        } else {
          stage(integral_constant<int, 0>{}, st, sK0, sV0, sK1, sV1);
          stage(integral_constant<int, 1>{}, st + 1, sK1, sV1, sK0, sV0);
          stage(integral_constant<int, 2>{}, st + 2, sK0, sV0, sK1, sV1);
          stage(integral_constant<int, 3>{}, st + 3, sK1, sV1, sK0, sV0);
        }
      }
    }

    // The loads of the stages behind the end have landed: none is on its way to LDS when a workgroup ends, and another has its LDS.
    __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0)
    asm volatile("" : : : "memory");

    const bool whole = first == 0 && stages == s.blocks;   // the tile is this worker's alone
    {
    const int lane = fresh(tid & 63), lr = lane & 15, lg = lane >> 4, row0 = wave * 16 * QT + lr;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const int row = row0 + 16 * t;
      const float l = group4_sum(l_run[t]);
      if (whole) {
        const float inv = l > 0.f ? 1.f / l : 0.f;
        const bool none = magnitude_bits(l) == 0;   // the row sees nothing: 0, whatever V holds in rows that it does not see
        const int j = (r0 + row) / group, h = kvh * group + (r0 + row) % group;
        S* const o = static_cast<S*>(p.o) + ((int64_t)(s.start + j) * p.H + h) * D;
#pragma unroll
        for (int d0 = 0; d0 < DT; d0 += 2) {
          if constexpr (sizeof(S) == 4) {
#pragma unroll
            for (int d = d0; d < d0 + 2; ++d) {
              const f32x4 x = none ? f32x4{0.f, 0.f, 0.f, 0.f} : acc[t][d] * inv;
              if (row < rows) *reinterpret_cast<f32x4*>(o + 16 * d + 4 * lg) = x;
            }
          } else {
            // lane groups lg and lg^1 trade halves so that each lane stores 8 consecutive channels
            u32x2 w[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              typedef S s4 __attribute__((ext_vector_type(4)));
              s4 a;
#pragma unroll
              for (int e = 0; e < 4; ++e) a[e] = (S)(none ? 0.f : acc[t][d0 + k][e] * inv);
              __builtin_memcpy(&w[k], &a, 8);
            }
            u32x4 x;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const auto y = __builtin_amdgcn_permlane16_swap(w[0][k], w[1][k], false, false);
              x[k] = y[0];
              x[2 + k] = y[1];
            }
            if (row < rows) *reinterpret_cast<u32x4*>(o + 16 * (d0 + (lg & 1)) + 4 * (lg & 2)) = x;
          }
        }
      } else if (row < rows) {
        // (the first piece of a share and its last one: no other piece is a part of a tile)
        const int64_t at_row = ((int64_t)(2 * worker + which) * p.Hkv + kvh) * ROWS + row;
        // (a maximum passes over NaN: a row whose logits are all NaN has sums all the same, NaN as its weights')
        const float m = m_run[t] == -INFINITY && magnitude_bits(l) > kInfBits ? 0.f : m_run[t];
        if (m > -INFINITY) {
#pragma unroll
          for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(p.sums + at_row * D + 16 * d + 4 * lg) = acc[t][d];
        }
        if (lg == 0) {
          p.stats[2 * at_row] = m;
          p.stats[2 * at_row + 1] = l;
        }
      }
    }
    // rows (bits) whose sums are not finite (a sum is not if a term is not) while their weights' sum is
    unsigned odd[QT], any = 0;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      f32x4 x = acc[t][0];
#pragma unroll
      for (int d = 1; d < DT; ++d) x += acc[t][d];
      const float sum = (x[0] + x[1]) + (x[2] + x[3]);
      const uint64_t bad = __builtin_amdgcn_ballot_w64(magnitude_bits(sum) >= kInfBits && row0 + 16 * t < rows);
      const uint64_t fine = __builtin_amdgcn_ballot_w64(magnitude_bits(group4_sum(l_run[t])) - 1u < kInfBits - 1u);
      odd[t] = (unsigned)((bad | bad >> 16 | bad >> 32 | bad >> 48) & fine) & 0xffffu;
      any |= odd[t];
    }
    if (any) {   // (uniform)
      __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): the rows as stored above come first
      asm volatile("" : : : "memory");
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const float l = group4_sum(l_run[t]);
        for (unsigned left = odd[t]; left; left &= left - 1) {
          const int i = __builtin_ctz(left), row = w0 + 16 * t + i, j = (r0 + row) / group, h = kvh * group + (r0 + row) % group;
          const float m = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(m_run[t]), i));
          const float li = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(l), i));
          void* const out = whole ? static_cast<void*>(static_cast<S*>(p.o) + ((int64_t)(s.start + j) * p.H + h) * D)
                                  : static_cast<void*>(p.sums + (((int64_t)(2 * worker + which) * p.Hkv + kvh) * ROWS + row) * D);
          tree_row_again<S, D>(p, s, b, kvh, h, j, seen_by(row), first * SR, end * SR < s.n ? end * SR : s.n, m, whole ? 1.f / li : 1.f,
                               out, whole, lane);
        }
      }
    }
    }
    if (p.direct) return;
    // the join's: the tile's first worker, how many have a part of it, and which piece the first one's is
    if (first == 0 && tid == 0 && kvh == 0) {
      int* const own = p.owners + 4 * ((int64_t)((s.start * group) >> LB) + b + tile);
      own[0] = worker;
      own[1] = (int)((before + s.blocks - 1) / size) - worker + 1;
      own[2] = which;
    }
    at += stages - first;
    if (at >= stop) return;
    before += s.blocks;
    first = 0;
    which = 1;
    if (++tile == s.tiles) {
      tile = 0;
      do {   // (stages are left, so a sequence with tokens follows)
        if (++b == p.B) return;
      } while (cu_at(p.cu, b + 1, p.T) <= cu_at(p.cu, b, p.T));
    }
    loads_barrier<0>();   // (the last stages have been read)
  }
}

// O of the tiles that more than one worker had a part of, and zeros of the tokens behind the last
// sequence.  A workgroup takes 16 rows of a tile; a thread 4 channels of one.
template <typename S, int D, int QT>
__global__ void __launch_bounds__(256) tree_join_kernel(const TreeParams p) {
  constexpr int ROWS = 64 * QT, LB = QT == 2 ? 7 : 6, SUB = ROWS / 16, Q = D / 4;
  const int tid = thread_id(), lane = tid & 63;
  const int sub = block_id() % SUB, rest = block_id() / SUB, kvh = rest % p.Hkv, slot = rest / p.Hkv, group = p.H / p.Hkv;
  int b, tile;
  find_rows(p, LB, slot, lane, b, tile);
  const int start = cu_at(p.cu, b, p.T), end = b < p.B ? cu_at(p.cu, b + 1, p.T) : p.T;
  const int rows = (end > start ? end - start : 0) * group - tile * ROWS;   // (of this tile and those behind it)
  if (rows <= 16 * sub) return;
  int w0 = 0, n = 0, which = 0;
  if (b < p.B) {
    w0 = p.owners[4 * (int64_t)slot];
    n = p.owners[4 * (int64_t)slot + 1];
    which = p.owners[4 * (int64_t)slot + 2];
    // finished by its worker; or, where starts do not ascend, no worker's
    if (n <= 1 || w0 < 0 || n > p.workers || w0 > p.workers - n || (which & ~1)) return;
  }
  for (int u = tid; u < 16 * Q; u += 256) {
    const int row = 16 * sub + u / Q, c = 4 * (u % Q);
    if (row >= rows) break;
    auto at = [&](int i) { return ((int64_t)(2 * (w0 + i) + (i ? 0 : which)) * p.Hkv + kvh) * ROWS + row; };
    float m = -INFINITY, l = 0.f;
    f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
    constexpr int PER = 4;   // parts whose loads are on their way together
    for (int i0 = 0; i0 < n; i0 += PER) {
      typedef float f2 __attribute__((ext_vector_type(2)));
      f2 st[PER];
      f32x4 y[PER];
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        const int64_t a = at(i0 + u < n ? i0 + u : n - 1);
        st[u] = *reinterpret_cast<const f2*>(p.stats + 2 * a);
        y[u] = *reinterpret_cast<const f32x4*>(p.sums + a * D + c);
      }
      float top = m;
#pragma unroll
      for (int u = 0; u < PER; ++u) top = fmaxf(top, st[u][0]);
      if (top == -INFINITY) continue;   // (such parts have seen nothing and have no sums)
      const float keep = m == -INFINITY ? 0.f : fmaxf(fast_exp2(m - top), 0x1p-126f);   // (an infinite sum stays one)
      l *= keep;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = m == -INFINITY ? 0.f : x[e] * keep;
      m = top;
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        const bool in = i0 + u < n && st[u][0] != -INFINITY;
        const float a = fmaxf(fast_exp2(st[u][0] - top), 0x1p-126f);
        l += in ? a * st[u][1] : 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += in ? a * y[u][e] : 0.f;
      }
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    const int r = tile * ROWS + row;
    const float y[4] = {x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv};
    store4<S>(static_cast<S*>(p.o) + ((int64_t)(start + r / group) * p.H + kvh * group + r % group) * D + c, 1, true, y);
  }
}

template <typename S, int D, int QT>
static hipError_t tree(const TreeParams& p, hipStream_t st) {
  constexpr int SUB = 4 * QT;
  hipLaunchKernelGGL((tree_kernel<S, D, QT>), dim3((unsigned)p.Hkv * (unsigned)(p.direct ? p.slots : p.workers)), dim3(kSeqThreads), 0, st, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.direct) return e;
  hipLaunchKernelGGL((tree_join_kernel<S, D, QT>), dim3((unsigned)p.slots * p.Hkv * SUB), dim3(256), 0, st, p);
  return hipGetLastError();
}
template <typename S, int D>
static hipError_t tree_rows(const TreeParams& p, hipStream_t st) {
  if constexpr (sizeof(S) == 2)
    if (p.rows == 128) return tree<S, D, 2>(p, st);
  return tree<S, D, 1>(p, st);
}
template <typename S>
static hipError_t tree_d(const TreeParams& p, int D, hipStream_t st) {
  return D == 32 ? tree_rows<S, 32>(p, st) : D == 64 ? tree_rows<S, 64>(p, st) : D == 128 ? tree_rows<S, 128>(p, st) : tree_rows<S, 256>(p, st);
}
hipError_t launch_tree(const TreeParams& p, int dt, int D, hipStream_t st) {
  return dt == DT_BF16 ? tree_d<bf16>(p, D, st) : dt == DT_F16 ? tree_d<f16>(p, D, st) : tree_d<float>(p, D, st);
}

}  // namespace farope
