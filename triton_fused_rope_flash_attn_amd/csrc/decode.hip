// Attention of one new token per sequence over its paged cache.
//
//   q-hat = R(position) q;  O = softmax(scale q-hat K^T) V over the sequence's cached rows
//   (K is cached rotated);  a sequence of no rows has O = 0.
//
// Bound by memory: the cache is read once.  A workgroup takes a part of one
// sequence's rows of one key head for up to 16 query heads of its group, which share
// them; each of its waves streams its own 32-row blocks of K and V to LDS (16 bytes
// per lane straight from their pages, double-buffered), with no barrier until the
// waves' sums are joined.  With more than one part, the parts' unnormalised sums go
// to the workspace and decode_join_kernel joins them.
//
// The products run on MFMA with the 16 query heads as columns.  Their rate is far
// from binding, so 16-bit tensors keep fp32 accuracy where it costs no memory: q-hat
// and P enter as a pair of 16-bit values (x = hi + lo), K and V are exact as cached.
#include <type_traits>

#include "seq.h"

namespace farope {

// Rows that do not exist (behind the sequence's end, on no page of the cache) are
// read from here, so that what the cache holds there does not matter.
static __device__ __align__(1024) const unsigned zero_row[256] = {};

template <typename S, int D> struct DecodeShape {
  static constexpr int RB = D * (int)sizeof(S);
  static constexpr int NW = RB <= 256 ? 4 : RB == 512 ? 2 : 1;   // waves: what LDS holds
};

// x = hi + lo in the operand type (fp32: hi alone)
template <typename S> struct Split {
  using C = typename SeqComp<S>::C;
  static constexpr bool kTwo = sizeof(S) == 2;
  typename C::Frag hi, lo;
  __device__ __forceinline__ void set(const float (&x)[8]) {
    hi = C::make(x);
    if constexpr (kTwo) {
      float r[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = x[e] - (float)hi.v[e];
      lo = C::make(r);
    }
  }
  __device__ __forceinline__ f32x4 mma(const typename C::Frag& a, f32x4 c) const {
    if constexpr (kTwo) c = C::mma(a, lo, c);
    return C::mma(a, hi, c);
  }
};

template <typename S, int D>
__global__ void __launch_bounds__((64 * DecodeShape<S, D>::NW)) decode_kernel(const DecodeParams p) {
  using T = Tile<S, D>;
  constexpr int NW = DecodeShape<S, D>::NW, KS = D / 32, DT = D / 16, BLK = 32 * D, NI = 32 / T::RPI;
  // per wave a K and a V block in each; afterwards the waves' sums [16][D] in the first
  __shared__ __attribute__((aligned(16))) S buf0[NW * 2 * BLK], buf1[NW * 2 * BLK];
  __shared__ float stat[NW][2][16];

  const int tid = thread_id();
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int lr = lane & 15, lg = lane >> 4;
  const int part = block_id() % p.parts, rest = block_id() / p.parts;
  const int gt = rest % p.g_tiles, bh = rest / p.g_tiles, b = bh / p.Hkv, kvh = bh % p.Hkv;
  const int group = p.H / p.Hkv, left = group - 16 * gt, nq = left < 16 ? left : 16;
  const int head0 = kvh * group + 16 * gt;

  // the sequence's rows, as far as its page list goes; this part's share, in whole blocks
  const int64_t room = (int64_t)p.c.max_pages * p.c.page;
  int len = p.c.lengths[b];
  len = len < 0 ? 0 : len > room ? (int)room : len;
  const int blocks = (len + 31) >> 5, share = (blocks + p.parts - 1) / p.parts;
  const int first = part * share, end = first + share < blocks ? first + share : blocks;

  // lane l (and l + 32): the page of row 32 blk + l, or -1, and the row within it
  const int* const pages = p.c.pages + b * p.c.spages;
  struct Ids { int page, row; };
  auto fetch = [&](int blk) __attribute__((always_inline)) {
    const int r = 32 * blk + (lane & 31);
    Ids id{-1, 0};
    if (blk < end && r < len) {
      const int place = (int)((unsigned)r / (unsigned)p.c.page);
      id.page = pages[place];
      id.row = r - place * p.c.page;
    }
    return id;
  };
  auto ptr = [&](const void* base, const int64_t* st, const Ids& id, int row) __attribute__((always_inline)) {
    const int g = __builtin_amdgcn_ds_bpermute(4 * row, id.page), r = __builtin_amdgcn_ds_bpermute(4 * row, id.row);
    const S* a = static_cast<const S*>(base) + g * st[0] + r * st[1] + kvh * st[2];
    return g < 0 || g >= p.c.n_pages ? reinterpret_cast<const S*>(zero_row) : a;
  };
  auto load = [&](S* kd, S* vd, const Ids& id) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < NI; ++g) {
      const int row = g * T::RPI + lane / T::CPR, ch = ((lane % T::CPR) ^ T::chunk_xor(row)) * T::EPC;
      seq_dma16(ptr(p.c.kc, p.c.skc, id, row) + ch, kd + g * T::RPI * D);
      seq_dma16(ptr(p.c.vc, p.c.svc, id, row) + ch, vd + g * T::RPI * D);
    }
  };

  // q-hat * scale * log2 e: column lr is query head head0 + lr (heads past the group: zeros)
  Split<S> qf[KS];
  {
    const int pos = p.positions ? p.positions[b] : len - 1 - p.has_cls;
    const int tr = table_row(pos, p.n_pos);
    const S* qp = static_cast<const S*>(p.q) + b * p.sq[0] + (head0 + (lr < nq ? lr : 0)) * p.sq[1];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float x[8], cs[8];
      row8<S>(qp + (32 * s + 8 * lg) * p.sq[2], p.sq[2], p.vec_q, x);
      table_load4(p.cosp, p.sinp, tr, D / 2, 16 * s + 4 * lg, cs);
      rope_rotate8(x, cs);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = lr < nq ? x[e] * p.c2 : 0.f;
      qf[s].set(x);
    }
  }
  f32x4 acc[DT];
  float m_run = -INFINITY, l_run = 0.f, thr = -INFINITY;
  f32x4 nm4 = f32x4{0.f, 0.f, 0.f, 0.f};   // minus the running max (0 before the first row)
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  FragAt<S, D> at;
  at.init(lr, lg);

  auto block = [&](const S* __restrict__ k, const S* __restrict__ v, unsigned rows) __attribute__((always_inline)) {
    f32x4 sacc[2];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) sacc[h] = qf[s].mma(at.row(k, s, h), s == 0 ? nm4 : sacc[h]);
    if (rows != 0xffffffffu) {   // uniform: rows (bits) that do not exist
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) sacc[h][i] = rows >> (16 * h + 4 * lg + i) & 1 ? sacc[h][i] : -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int h = 0; h < 2; ++h) mx = fmaxf(mx, fmaxf(fmaxf(sacc[h][0], sacc[h][1]), fmaxf(sacc[h][2], sacc[h][3])));
    if (__any(mx > thr)) {   // (as in the forward over packed sequences)
      thr = 8.0f;
      const float old = m_run == -INFINITY ? 0.f : m_run;
      const float mnew = fmaxf(m_run, group4_max(mx) + old);
      const float alpha = fast_exp2(m_run - mnew), sh = old - mnew;
      m_run = mnew;
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d] *= alpha;
#pragma unroll
      for (int h = 0; h < 2; ++h) sacc[h] += sh;
      nm4 = f32x4{-mnew, -mnew, -mnew, -mnew};
    }
    float x[8];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * h + i] = fast_exp2(sacc[h][i]);
    l_run += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
    Split<S> pf;
    pf.set(x);
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = pf.mma(at.col(v, d), acc[d]);
  };

  // block i of the wave is first + wave + NW i; page ids are fetched two blocks
  // ahead, rows one
  auto valid = [&](const Ids& id) __attribute__((always_inline)) {
    return (unsigned)__builtin_amdgcn_ballot_w64(id.page >= 0 && id.page < p.c.n_pages);
  };
  int blk = first + wave;
  Ids id0 = fetch(blk), id1 = fetch(blk + NW);
  S* const mine0 = buf0 + wave * 2 * BLK;
  S* const mine1 = buf1 + wave * 2 * BLK;
  auto step = [&](S* __restrict__ cur, S* __restrict__ next) __attribute__((always_inline)) {
    const unsigned rows = valid(id0);
    id0 = id1;
    id1 = fetch(blk + 2 * NW);
    wave_lds_reads_done();
    if (blk + NW < end) {
      load(next, next + BLK, id0);
      wave_lds_fence();
      __builtin_amdgcn_s_waitcnt(vm_wait(2 * NI));   // all but the loads just issued have landed
    } else {
      __builtin_amdgcn_s_waitcnt(vm_wait(0));
    }
    wave_lds_fence();
    block(cur, cur + BLK, rows);
    blk += NW;
  };
  if (blk < end) load(mine0, mine0 + BLK, id0);
  while (blk < end) {
    step(mine0, mine1);
    if (blk >= end) break;
    step(mine1, mine0);
  }

  // join the waves: m = max, l and O rescaled to it
  const float l = group4_sum(l_run);
  if (lg == 0) {
    stat[wave][0][lr] = m_run;
    stat[wave][1][lr] = l;
  }
  lds_barrier();
  float m = -INFINITY;
#pragma unroll
  for (int w = 0; w < NW; ++w) m = fmaxf(m, stat[w][0][lr]);
  const float mine_scale = m_run == -INFINITY ? 0.f : fast_exp2(m_run - m);
  float* const sums = reinterpret_cast<float*>(buf0);
  constexpr int WS = 2 * BLK * (int)sizeof(S) / 4;   // a wave's own part, which it has read: 16 D floats fit
  float* const out = sums + wave * WS + lr * D;
#pragma unroll
  for (int d = 0; d < DT; ++d) {
    const f32x4 x = acc[d] * mine_scale;
    *reinterpret_cast<f32x4*>(out + 16 * d + 4 * lg) = x;
  }
  lds_barrier();
  for (int i = tid; i < nq * (D / 8); i += 64 * NW) {
    const int q = i / (D / 8), c = 8 * (i % (D / 8));
    float mq = -INFINITY, lq = 0.f, x[8] = {};
#pragma unroll
    for (int w = 0; w < NW; ++w) mq = fmaxf(mq, stat[w][0][q]);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float mw = stat[w][0][q];
      lq += mw == -INFINITY ? 0.f : stat[w][1][q] * fast_exp2(mw - mq);
      const float* y = sums + w * WS + q * D + c;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] += y[e];
    }
    const int64_t row = (int64_t)b * p.H + head0 + q;
    if (p.parts == 1) {
      const float inv = lq > 0.f ? 1.f / lq : 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= inv;
      put_row8<S>(static_cast<S*>(p.o) + row * D + c, x);
    } else {
      put_row8<float>(p.sums + (row * p.parts + part) * D + c, x);
      if (c == 0) {
        p.stats[(row * p.parts + part) * 2] = mq;
        p.stats[(row * p.parts + part) * 2 + 1] = lq;
      }
    }
  }
}

// O of the parts' sums: a thread takes 4 channels of one (sequence, query head).
template <typename S, int D>
__global__ void __launch_bounds__(256) decode_join_kernel(const DecodeParams p) {
  const int64_t i = (int64_t)block_id() * 256 + thread_id(), row = i / (D / 4);
  const int c = 4 * (int)(i % (D / 4));
  if (row >= (int64_t)p.B * p.H) return;
  const float* const st = p.stats + row * p.parts * 2;
  float m = -INFINITY;
  for (int s = 0; s < p.parts; ++s) m = fmaxf(m, st[2 * s]);
  float l = 0.f;
  f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < p.parts; ++s) {
    if (st[2 * s] == -INFINITY) continue;   // (no rows in this part)
    const float a = fast_exp2(st[2 * s] - m);
    l += a * st[2 * s + 1];
    x += a * *reinterpret_cast<const f32x4*>(p.sums + (row * p.parts + s) * D + c);
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  const float y[4] = {x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv};
  store4<S>(static_cast<S*>(p.o) + row * D + c, 1, true, y);
}

template <typename S, int D>
static hipError_t decode(const DecodeParams& p, hipStream_t st) {
  constexpr int NW = DecodeShape<S, D>::NW;
  hipLaunchKernelGGL((decode_kernel<S, D>), dim3((unsigned)(p.B * p.Hkv * p.g_tiles * p.parts)), dim3(64 * NW), 0, st, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.parts == 1) return e;
  const int64_t n = (int64_t)p.B * p.H * (D / 4);
  hipLaunchKernelGGL((decode_join_kernel<S, D>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, p);
  return hipGetLastError();
}
template <typename S>
static hipError_t decode_d(const DecodeParams& p, int D, hipStream_t st) {
  return D == 32 ? decode<S, 32>(p, st) : D == 64 ? decode<S, 64>(p, st) : D == 128 ? decode<S, 128>(p, st) : decode<S, 256>(p, st);
}
hipError_t launch_decode(const DecodeParams& p, int dt, int D, hipStream_t st) {
  return dt == DT_BF16 ? decode_d<bf16>(p, D, st) : dt == DT_F16 ? decode_d<f16>(p, D, st) : decode_d<float>(p, D, st);
}

}  // namespace farope
