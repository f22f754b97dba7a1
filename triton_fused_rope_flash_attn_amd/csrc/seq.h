// Packed sequences: what the kernels of attention over sequences of different
// lengths share (seq_prep.hip, seq_fwd.hip, seq_bwd.hip, cache.hip, decode.hip).
//
// T tokens of B sequences lie behind each other; cu[0 .. B] are the sequences'
// first tokens and the end of the last one.  Tokens from cu[B] on belong to no
// sequence.  Tensors are [T, heads, D]; H query heads share Hkv key heads, query
// head h reads key head h / (H / Hkv).
#pragma once

#include "common.h"
#include "seq_params.h"

namespace farope {

// ---------------------------------------------------------------------------
// Operand types.  16-bit tensors are computed in their own type.  fp32 tensors
// are computed in fp32: v_mfma_f32_16x16x4_f32, whose lane group lg holds one
// contraction index per instruction, so eight of them take the same operand
// layout (8 values per lane) as one 16-bit instruction.
// ---------------------------------------------------------------------------
struct CompF32x {
  typedef float S;
  struct Frag { float v[8]; };
  static __device__ __forceinline__ Frag make(const float (&x)[8]) {
    Frag f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = x[e];
    return f;
  }
  static __device__ __forceinline__ Frag lds(const float* p) {
    Frag f;
    __builtin_memcpy(&f.v[0], __builtin_assume_aligned(p, 16), 32);
    return f;
  }
  static __device__ __forceinline__ f32x4 mma(const Frag& a, const Frag& b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[e], b.v[e], c, 0, 0, 0);
    return c;
  }
};
template <typename S> struct SeqComp;
template <> struct SeqComp<bf16> { using C = Comp<DT_BF16>; };
template <> struct SeqComp<f16> { using C = Comp<DT_F16>; };
template <> struct SeqComp<float> { using C = CompF32x; };

// Magnitude bits of x; 0x7f800000 and up are infinities and NaN.  (The kernels are compiled without
// regard for NaN: the empty asm keeps the compiler from concluding that x is none.)
__device__ __forceinline__ unsigned magnitude_bits(float x) {
  unsigned u = __float_as_uint(x);
  asm volatile("" : "+v"(u));
  return u & 0x7fffffffu;
}
constexpr unsigned kInfBits = 0x7f800000u;

// ---------------------------------------------------------------------------
// Softmax weights as operands of a product: P = exp2(s - m).  m is the row's running maximum, raised when a
// logit passes it by kSeqSlack (log2 units).  fp16 rounds what is below 2^-25 to 0, and a key of a row of 2^17 that
// far below the largest still counts in their sum (O of a row whose other keys weigh 2^-25 each was off
// by 3.9e-3).  There m is kept kWeightUp below the maximum: P up to 2^7, 2^15 before m is raised, and down to 2^-32 of
// the largest.  The weights of the backward are at most 1, and carry 2^kWeightUp alike.
// ---------------------------------------------------------------------------
template <typename S> constexpr float kWeightUp = std::is_same<S, f16>::value ? 7.0f : 0.0f;
constexpr float kSeqSlack = 8.0f;

// ---------------------------------------------------------------------------
// Streamed tiles: rows of D elements, unpadded, their 16-byte chunks XOR-swizzled
// per row with period 16 (as in stream.h: 16-byte reads of 16 rows and the
// transposed reads are free of bank conflicts).  A stage holds SR rows; a
// 16-byte-per-lane load to LDS fills RPI of them.
// ---------------------------------------------------------------------------
template <typename S, int D> constexpr int kStageRowsOf = D * sizeof(S) <= 256 ? 64 : 32;
template <typename S, int D, int ROWS = kStageRowsOf<S, D>> struct Tile {
  static constexpr int ES = sizeof(S), RB = D * ES, CPR = RB / 16, EPC = 16 / ES;
  static constexpr int SR = ROWS;
  static constexpr int RPI = CPR >= 64 ? 1 : 64 / CPR;
  static constexpr int NI = SR / (kSeqNW * RPI);      // loads per wave and stage
  static constexpr bool kSame = (kSeqNW * RPI) % 16 == 0;   // one swizzle pattern for all of them
  static __device__ __forceinline__ int chunk_xor(int r) {
    if constexpr (RB >= 256) return ((r >> 1) & 7) << 1;
    else if constexpr (ES == 4) return ((r >> 1) & 3) << 1;   // (pairs of chunks stay adjacent)
    else if constexpr (RB == 128) return ((((r >> 1) & 3) ^ ((r >> 2) & 2)) << 1) | ((r >> 3) & 1);
    else return (r >> 2) & 3;
  }
  static __device__ __forceinline__ int at(int r, int col) {
    return r * D + (((col / EPC) ^ chunk_xor(r)) * EPC) + (col % EPC);
  }
};

template <typename S, int D, int ROWS = kStageRowsOf<S, D>> struct SeqStream {
  using T = Tile<S, D, ROWS>;
  __amdgpu_buffer_rsrc_t rs;
  unsigned voff[T::kSame ? 1 : T::NI];
  unsigned row_b;     // bytes between rows
  // lane offsets; the rows' bytes are row_b apart
  __device__ __forceinline__ void lanes(int64_t stride, int wave, int lane) {
    row_b = (unsigned)stride * T::ES;
#pragma unroll
    for (int g = 0; g < (T::kSame ? 1 : T::NI); ++g) {
      const int r = (g * kSeqNW + wave) * T::RPI + lane / T::CPR;
      voff[g] = (unsigned)r * row_b + (unsigned)(((lane % T::CPR) ^ T::chunk_xor(r)) * 16);
    }
  }
  // rows [0, n) of a sequence's head; rows from n on read as zeros (unless rows overlap)
  __device__ __forceinline__ void base(const S* p, int n) {
    rs = make_rsrc(p, n > 0 ? (unsigned)(n - 1) * row_b + (unsigned)T::RB : 0u);
  }
  __device__ __forceinline__ void load(S* dst, int wave, int row0) const {
#pragma unroll
    for (int g = 0; g < T::NI; ++g) {
      if constexpr (T::kSame)
        lds_dma16(rs, dst + (wave + g * kSeqNW) * T::RPI * D, voff[0], (unsigned)(row0 + g * kSeqNW * T::RPI) * row_b);
      else
        lds_dma16(rs, dst + (wave + g * kSeqNW) * T::RPI * D, voff[g], (unsigned)row0 * row_b);
    }
  }
};

// 4 bytes per lane from a buffer straight into LDS (lane l lands at lds + 4 l).
__device__ __forceinline__ void seq_dma4(__amdgpu_buffer_rsrc_t r, void* lds, unsigned voff, unsigned soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 4, voff, soff, 0, 0);
}
// This wave's LDS loads have landed, and so have every wave's behind the barrier.
__device__ __forceinline__ void seq_stage_barrier() {
  __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0)
  lds_barrier();
}

// Operand fragments of a 32-row block of a staged tile: rows (row 16 h + lr, 8
// channels 32 s + 8 lg) and columns (channel 16 d + lr of the rows that output
// rows 4 lg + i of both halves are: k-slot 4 h + i is row 16 h + 4 lg + i).
template <typename S, int D> struct FragAt {
  using C = typename SeqComp<S>::C;
  using T = Tile<S, D>;
  // Column reads: 16 bits, each tile's own; fp32, of rows 4 lg and 4 lg + 2 and the first four
  // tiles: the swizzle is the same for the row behind an even one, for rows 16 apart and for
  // tiles 4 apart (it moves chunks within 16), which are then constant steps.  (Held apart, each
  // tile's and row's, they filled the registers: decode of 16 x 4096 rows, 2 key heads, D 256 126 us
  // instead of 82; forward and backward of 51 x 290 tokens, 48 heads, D 128 1253 instead of 1140.)
  static constexpr int NT = sizeof(S) == 2 ? D / 16 : D / 16 < 4 ? D / 16 : 4, NR = sizeof(S) == 2 ? 1 : 2;
  int ao[D / 32], to[NT][NR];
  __device__ __forceinline__ void init(int lr, int lg) {
#pragma unroll
    for (int s = 0; s < D / 32; ++s) ao[s] = T::at(lr, 32 * s + 8 * lg);
#pragma unroll
    for (int d = 0; d < NT; ++d)
#pragma unroll
      for (int r = 0; r < NR; ++r)
        to[d][r] = sizeof(S) == 2 ? T::at(4 * lg + (lr >> 2), 16 * d + 4 * (lr & 3)) : T::at(4 * lg + 2 * r, 16 * d + lr);
  }
  __device__ __forceinline__ typename C::Frag row(const S* block, int s, int h) const {
    return C::lds(block + ao[s] + 16 * h * D);
  }
  __device__ __forceinline__ typename C::Frag col(const S* block, int d) const {
    if constexpr (sizeof(S) == 2) {
      return C::tr(block + to[d][0], block + to[d][0] + 16 * D);
    } else {
      typename C::Frag f;
#pragma unroll
      for (int e = 0; e < 8; ++e) f.v[e] = block[to[d & 3][(e >> 1) & 1] + (16 * (e >> 2) + (e & 1)) * D + 64 * (d >> 2)];
      return f;
    }
  }
};

// ---------------------------------------------------------------------------
// Sequences and tiles.  Values of cu are clamped to [0, T], so no value of them
// takes an access outside the tensors.
// ---------------------------------------------------------------------------
__device__ __forceinline__ int cu_at(const int* __restrict__ cu, int i, int T) {
  const int x = i == 0 ? 0 : cu[i];
  return x < 0 ? 0 : x > T ? T : x;
}

struct SeqTile {
  int seq;      // B: the tokens behind the last sequence
  int start;    // first token of the sequence
  int len;      // its tokens
  int tile;     // tile of this workgroup within it (< 0: none)
  int tiles;    // its tiles
};

// Workgroups come as slots of 2^lb rows: sequence i takes slots (cu[i] >> lb) + i on,
// at least as many as it has tiles, so the grid needs T and B alone: no length
// crosses to the host.  All 64 lanes search together (64 boundaries a step).
__device__ __forceinline__ SeqTile find_tile(const int* __restrict__ cu, int B, int T, int lb, int slot, int lane) {
  int lo = 0, n = B + 1;
  while (n > 1) {
    const int step = (n + 63) >> 6, j = lane * step;
    const bool le = j < n && (cu_at(cu, lo + (j < n ? j : 0), T) >> lb) + lo + j <= slot;
    const int k = 63 - __builtin_clzll(__builtin_amdgcn_ballot_w64(le) | 1ull);
    lo += k * step;
    n = n - k * step < step ? n - k * step : step;
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  SeqTile t;
  t.seq = lo;
  t.start = cu_at(cu, lo, T);
  const int end = lo < B ? cu_at(cu, lo + 1, T) : T;
  t.len = end > t.start ? end - t.start : 0;
  t.tiles = (t.len + (1 << lb) - 1) >> lb;
  t.tile = slot - ((t.start >> lb) + lo);
  if (t.tile >= t.tiles) t.tile = -1;
  return t;
}
// Inclusive sums over the wave's lanes: DPP shifts within each row of 16 lanes, then the
// last lane of a row, and of half the wave, added to the rows behind.
__device__ __forceinline__ unsigned wave_scan(unsigned x) {
  x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xF, 0xF, false);   // row_shr 1, 2, 4, 8
  x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xF, 0xF, false);
  x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xF, 0xF, false);
  x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xF, 0xF, false);
  x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xA, 0xF, false);   // row_bcast 15, 31
  x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xC, 0xF, false);
  return x;
}

// The same, causal, in the order of the tiles' work: the r-th heaviest tile of the call for
// r = slot (then the tokens behind the last sequence).  Level l holds the tiles with l
// tiles of their sequence's keys before them (of its queries behind them: `keys`), one of
// each sequence of more than l tiles.  The workgroups that start last are then the short ones.
__device__ __forceinline__ SeqTile ordered_tile(const int* __restrict__ cu, int B, int T, int lb, int slot, int lane, bool keys) {
  int nt[kOrderSeqs / 64];
#pragma unroll
  for (int k = 0; k < kOrderSeqs / 64; ++k) {
    nt[k] = 0;
    if (64 * k >= B) continue;
    const int i = 64 * k + lane;
    if (i < B) {
      const int n = cu_at(cu, i + 1, T) - cu_at(cu, i, T);
      nt[k] = n > 0 ? (n + (1 << lb) - 1) >> lb : 0;
    }
  }
  auto from = [&](int l) {   // tiles of levels l and up
    unsigned n = 0;
#pragma unroll
    for (int k = 0; k < kOrderSeqs / 64; ++k) n += nt[k] > l ? (unsigned)(nt[k] - l) : 0u;
    return __builtin_amdgcn_readlane((int)wave_scan(n), 63);
  };
  SeqTile t;
  const int tiles = from(0);
  if (slot >= tiles) {
    t.seq = B;
    t.start = cu_at(cu, B, T);
    t.len = T - t.start;
    t.tiles = (t.len + (1 << lb) - 1) >> lb;
    t.tile = slot - tiles < t.tiles ? slot - tiles : -1;
    return t;
  }
  int l = 0, above = 0;   // the largest level l with from(l) > slot; above = from(l + 1)
  for (int hi = tiles; hi - l > 1;) {
    const int mid = (l + hi) >> 1, n = from(mid);
    if (n > slot) l = mid; else { hi = mid; above = n; }
  }
  int j = slot - above;
  t.seq = 0;
#pragma unroll
  for (int k = 0; k < kOrderSeqs / 64; ++k) {
    const uint64_t m = __builtin_amdgcn_ballot_w64(nt[k] > l);
    const int n = __builtin_popcountll(m);
    if (j >= 0 && j < n) {
      const int below = __builtin_amdgcn_mbcnt_hi((unsigned)(m >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)m, 0u));
      t.seq = 64 * k + __builtin_ctzll(__builtin_amdgcn_ballot_w64((m >> lane & 1) && below == j));
      t.tiles = __builtin_amdgcn_readlane(nt[k], t.seq & 63);
    }
    j -= n;
  }
  t.start = cu_at(cu, t.seq, T);
  const int end = cu_at(cu, t.seq + 1, T);
  t.len = end > t.start ? end - t.start : 0;
  t.tile = keys ? t.tiles - 1 - l : l;
  return t;
}
// A workgroup's tile of queries (keys: of keys), the later ones first (the earlier), which
// have more to do in a causal call: from the map that seq_prep_kernel has made, where
// there is such a pass, so that the heads' workgroups of a slot read 16 bytes instead of
// searching.
__device__ __forceinline__ SeqTile slot_tile(const SeqParams& p, int lb, int slot, int lane, bool keys) {
  const int* const map = keys ? p.map_k : p.map_q;
  if (!map) return find_tile(p.cu, p.B, p.T, lb, keys ? slot : p.slots - 1 - slot, lane);
  typedef int i4 __attribute__((ext_vector_type(4)));
  const i4 m = reinterpret_cast<const i4*>(map)[slot];
  SeqTile t;
  t.seq = __builtin_amdgcn_readfirstlane(m[0]);
  t.start = __builtin_amdgcn_readfirstlane(m[1]);
  t.len = __builtin_amdgcn_readfirstlane(m[2]);
  t.tile = __builtin_amdgcn_readfirstlane(m[3]);
  t.tiles = (t.len + (1 << lb) - 1) >> lb;
  return t;
}
// Sequence of token t (B: none), for the 64 lanes of a wave whose tokens are near each other.
__device__ __forceinline__ int find_seq(const int* __restrict__ cu, int B, int T, int first, int t, int lane) {
  int lo = 0, n = B + 1;
  while (n > 1) {
    const int step = (n + 63) >> 6, j = lane * step;
    const bool le = j < n && cu_at(cu, lo + (j < n ? j : 0), T) <= first;
    const int k = 63 - __builtin_clzll(__builtin_amdgcn_ballot_w64(le) | 1ull);
    lo += k * step;
    n = n - k * step < step ? n - k * step : step;
  }
  while (lo < B && cu_at(cu, lo + 1, T) <= t) ++lo;
  return lo;
}

// Table row of a token: `index` within its sequence, or the caller's position.  The
// class token (has_cls, index 0) and negative positions are not rotated (row -1);
// rows past the table take its last one.
__device__ __forceinline__ int table_row(int index, int n_pos) { return index < n_pos ? index : n_pos - 1; }

// cos and sin of pairs p0 .. p0 + 3 of a table row as rope_rotate8 takes them
__device__ __forceinline__ void table_load4(const float* __restrict__ cosp, const float* __restrict__ sinp, int row, int d2,
                                            int p0, float (&cs)[8]) {
  if (row < 0) {
#pragma unroll
    for (int p = 0; p < 4; ++p) { cs[2 * p] = 1.f; cs[2 * p + 1] = 0.f; }
    return;
  }
  const int64_t at = (int64_t)row * d2 + p0;
  const f32x4 c = *reinterpret_cast<const f32x4*>(cosp + at), s = *reinterpret_cast<const f32x4*>(sinp + at);
#pragma unroll
  for (int p = 0; p < 4; ++p) { cs[2 * p] = c[p]; cs[2 * p + 1] = s[p]; }
}

// 8 channels to a staged tile (one or two 16-byte chunks)
template <typename S, int D>
__device__ __forceinline__ void put_tile8(S* tile, int r, int col, const float (&x)[8]);

// 8 channels to a contiguous row (16 or 32 bytes)
template <typename S>
__device__ __forceinline__ void put_row8(S* __restrict__ p, const float (&x)[8]) {
  if constexpr (sizeof(S) == 4) {
    f32x4 a, b;
#pragma unroll
    for (int e = 0; e < 4; ++e) { a[e] = x[e]; b[e] = x[4 + e]; }
    reinterpret_cast<f32x4*>(p)[0] = a;
    reinterpret_cast<f32x4*>(p)[1] = b;
  } else {
    typedef S v8 __attribute__((ext_vector_type(8)));
    v8 a;
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = (S)x[e];
    *reinterpret_cast<v8*>(p) = a;
  }
}

template <typename S, int D>
__device__ __forceinline__ void put_tile8(S* tile, int r, int col, const float (&x)[8]) {
  put_row8<S>(tile + Tile<S, D>::at(r, col), x);   // (fp32: pairs of chunks stay adjacent)
}

// K rows rotated on their way to LDS: a thread loads its 8-channel pieces of a stage and
// their table entries early, and turns and stores them when the stage before has been
// read.  For short sequences, whose rows few workgroups read: it takes the place of
// seq_prep_kernel, whose launch and traffic they would notice.
template <typename S, int D, int ROWS = kStageRowsOf<S, D>> struct RotStage {
  using T = Tile<S, D, ROWS>;
  static constexpr int PPR = D / 8, N = T::SR * PPR / kSeqThreads;
  Raw8<S> raw[N];
  float cs[N][8];
  __device__ __forceinline__ void load(const SeqParams& p, const SeqTile& tl, int kvh, int st, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = st * T::SR + (tid + kSeqThreads * i) / PPR, c = 8 * (tid % PPR);
      const int rc = r < tl.len ? r : tl.len - 1;   // (keys past the end are masked)
      const int64_t tok = tl.start + rc;
      raw[i] = load_raw8<S>(static_cast<const S*>(p.k) + tok * p.sk[0] + kvh * p.sk[1] + c * p.sk[2], p.sk[2], p.vec_k);
      table_load4(p.cosp, p.sinp, table_row(p.positions ? p.positions[tok] : rc - p.has_cls, p.n_pos), D / 2, c / 2, cs[i]);
    }
  }
  __device__ __forceinline__ void store(const SeqParams& p, S* dst, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float x[8];
      unpack8(raw[i], x);
      rope_rotate8(x, cs[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= p.c2;
      put_tile8<S, D>(dst, (tid + kSeqThreads * i) / PPR, 8 * (tid % PPR), x);
    }
  }
};

}  // namespace farope
