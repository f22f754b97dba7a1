// Attention of one new token per sequence over its paged cache.
//
//   q-hat = R(position) q;  O = softmax(scale q-hat K^T) V over the sequence's cached rows
//   (K is cached rotated);  a sequence of no rows has O = 0.
//
// Bound by memory: the cache is read once.  The rows of all sequences, in blocks of
// 32, are divided evenly over the workers (workgroups) of a key head, whatever the
// sequences' lengths: a worker's share may end inside a sequence and run on in the
// next.  Up to 16 query heads of the key head's group share the rows.  A sequence
// that lies in one worker's share is finished there; of the others the workers leave
// unnormalised sums, which decode_join_kernel joins.
//
// The products run on MFMA with the 16 query heads as columns.  Their rate is far
// from binding, so 16-bit tensors keep fp32 accuracy where it costs no memory: q-hat
// and P enter as a pair of 16-bit values (x = hi + lo), K and V are exact as cached.
//
// Measured (us a call, both launches; bf16, D 128): 2 sequences up to 100000 rows, 8 key heads
// 119 (5.2 TB/s of cache), 48 up to 4097, 4 key heads 45 (3.7 TB/s: the kernel 35, the join 5, the
// step between them); 1 sequence of 197 rows, 12 heads, D 64 6.8, one round of memory latency
// and the launch; fp32, 5 up to 1025, 8 heads, D 64 13.3, two launches.
#include <type_traits>

#include "seq.h"

namespace farope {

constexpr int kDecodeNW = 4;   // waves per worker, which take its blocks in turn

// x = hi + lo in the operand type (fp32: hi alone).  hi lies nearer to 0 than x, so that lo has its sign and is
// not 0: the two products with an infinity of K or V then are the infinity that x times it is, not a NaN.  (Up
// to what fp16 rounds to 0: weights of 2^-31 of the largest.)
template <typename S> struct Split {
  using C = typename SeqComp<S>::C;
  static constexpr bool kTwo = sizeof(S) == 2;
  typename C::Frag hi, lo;
  __device__ __forceinline__ void set(const float (&x)[8]) {   // (no -0)
    if constexpr (!kTwo) {
      hi = C::make(x);
      return;
    }
    float h[8], r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float below = __uint_as_float(__builtin_elementwise_sub_sat(__float_as_uint(x[e]), 1u));
      if constexpr (std::is_same<S, f16>::value) h[e] = (float)__builtin_amdgcn_cvt_pkrtz(below, 0.f)[0];
      else h[e] = __uint_as_float(__float_as_uint(below) & 0xffff0000u);
      r[e] = x[e] - h[e];
      if constexpr (std::is_same<S, f16>::value) {   // at least fp16's least value
        const float least = __builtin_amdgcn_fmed3f(x[e], -0x1p-24f, 0x1p-24f);
        r[e] = fabsf(r[e]) < fabsf(least) ? least : r[e];
      }
    }
    hi = C::make(h);   // (exact)
    lo = C::make(r);
  }
  __device__ __forceinline__ f32x4 mma(const typename C::Frag& a, f32x4 c) const {
    if constexpr (kTwo) c = C::mma(a, lo, c);
    return C::mma(a, hi, c);
  }
};

// Rows of sequence b, as far as its page list goes, and their blocks of 32.
__device__ __forceinline__ int cached_rows(const DecodeParams& p, int b) {
  const int64_t room = (int64_t)p.c.max_pages * p.c.page;
  const int len = p.c.lengths[b];
  return len < 0 ? 0 : len > room ? (int)room : len;
}
__device__ __forceinline__ int cached_blocks(const DecodeParams& p, int b) { return (int)(((int64_t)cached_rows(p, b) + 31) >> 5); }

__device__ __forceinline__ int64_t shfl64(int64_t x, int lane) {
  const int lo = __builtin_amdgcn_ds_bpermute(4 * lane, (int)x), hi = __builtin_amdgcn_ds_bpermute(4 * lane, (int)(x >> 32));
  return (int64_t)((uint64_t)(unsigned)hi << 32 | (unsigned)lo);
}
template <typename S, int D>
__global__ void __launch_bounds__(64 * kDecodeNW, D * sizeof(S) <= 128 ? 3 : D * sizeof(S) <= 256 ? 2 : 1) decode_kernel(const DecodeParams p) {
  using T = Tile<S, D>;
  using Frag = typename SeqComp<S>::C::Frag;
  constexpr int NW = kDecodeNW, KS = D / 32, DT = D / 16, BLK = 32 * D, VJ = T::CPR / 4;
  typedef Raw8<S> K8;
  typedef u32x4 V16;
  // per wave its V block; afterwards its sums [16][D]
  __shared__ __attribute__((aligned(16))) S buf[NW * BLK];
  __shared__ float stat[NW][2][16];

  const int tid = thread_id();
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int lr = lane & 15, lg = lane >> 4;
  const int heads = p.Hkv * p.g_tiles, worker = block_id() / heads, hx = block_id() % heads;
  const int kvh = hx / p.g_tiles, gt = hx % p.g_tiles;
  const int group = p.H / p.Hkv, left = group - 16 * gt, nq = left < 16 ? left : 16;
  const int head0 = kvh * group + 16 * gt;

  // this worker's blocks [at, stop) of all, from block `first` of sequence b on; `before`
  // are the blocks of the sequences before b
  int b = worker, first = 0;
  int64_t at = 0, stop = 0, before = 0, size = 1;
  if (!p.direct) {
    int64_t all = 0;
    unsigned n = 0, sum = 0;
    for (int i = 0; i < p.B; i += 64) {   // (blocks of 64 sequences: less than 2^32)
      n = i + lane < p.B ? (unsigned)cached_blocks(p, i + lane) : 0u;
      sum = wave_scan(n);
      all += (unsigned)__builtin_amdgcn_readlane((int)sum, 63);
    }
    const int64_t even = (all + p.workers - 1) / p.workers;
    size = even > kDecodeNW ? even : kDecodeNW;   // (a block for each wave at least)
    at = worker * size;
    if (at >= all) return;
    stop = at + size < all ? at + size : all;
    b = -1;
    for (int i = 0; i < p.B; i += 64) {   // (some sequence holds block `at`)
      if (p.B > 64) {
        n = i + lane < p.B ? (unsigned)cached_blocks(p, i + lane) : 0u;
        sum = wave_scan(n);
      }
      const uint64_t past = __builtin_amdgcn_ballot_w64(before + sum > at);
      if (past) {
        const int l = __builtin_ctzll(past);
        b = i + l;
        before += (unsigned)(__builtin_amdgcn_readlane((int)sum, l) - __builtin_amdgcn_readlane((int)n, l));
        break;
      }
      before += (unsigned)__builtin_amdgcn_readlane((int)sum, 63);
    }
    if (b < 0) return;
    first = (int)(at - before);
  }

  S* const vs = buf + wave * BLK;
  float* const sums = reinterpret_cast<float*>(buf);
  constexpr int WS = BLK * (int)sizeof(S) / 4;   // a wave's own part: 16 D floats fit
  FragAt<S, D> frag;
  frag.init(lr, lg);
  const int vrow = lane >> 2, vch = lane & 3;    // V chunks of a lane: rows vrow + 16 h, 16-byte chunks vch + 4 j

  for (;;) {
    const int len = cached_rows(p, b), blocks = (int)(((int64_t)len + 31) >> 5);
    const int end = p.direct || stop - at > blocks - first ? blocks : first + (int)(stop - at);

    // lane l (and l + 32): row 32 blk + l of the sequence: element offsets in the caches, whether it exists
    const int* const pages = p.c.pages + b * p.c.spages;
    struct Ids { int page, row; };
    auto fetch = [&](int blk) __attribute__((always_inline)) {
      Ids id{-1, 0};
      if (blk < end) {
        const unsigned r = 32u * (unsigned)blk + (unsigned)(lane & 31);
        if (r < (unsigned)len) {
          const unsigned place = r / (unsigned)p.c.page;
          id.page = pages[place];
          id.row = (int)(r - place * (unsigned)p.c.page);
        }
      }
      return id;
    };
    K8 kr[2][KS];
    V16 vr[2][VJ];
    unsigned rows = 0;   // rows (bits) of the loaded block that exist; the others read page 0's first row
    auto load = [&](const Ids& id) __attribute__((always_inline)) {
      const bool in = id.page >= 0 && id.page < p.c.n_pages;
      rows = (unsigned)__builtin_amdgcn_ballot_w64(in);
      const int64_t g = in ? id.page : 0, r = in ? id.row : 0;
      const int64_t ko = g * p.c.skc[0] + r * p.c.skc[1], vo = g * p.c.svc[0] + r * p.c.svc[1];
      const S* const kb = static_cast<const S*>(p.c.kc) + kvh * p.c.skc[2] + 8 * lg;
      const S* const vb = static_cast<const S*>(p.c.vc) + kvh * p.c.svc[2] + vch * T::EPC;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const S* const kp = kb + shfl64(ko, 16 * h + lr);
#pragma unroll
        for (int s = 0; s < KS; ++s) kr[h][s] = load_raw8<S>(kp + 32 * s, 1, true);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const S* const vp = vb + shfl64(vo, 16 * h + vrow);
#pragma unroll
        for (int j = 0; j < VJ; ++j) vr[h][j] = *reinterpret_cast<const V16*>(vp + 4 * j * T::EPC);
      }
    };
    // block i of the wave is first + wave + NW i; page numbers are read two blocks
    // ahead, rows one
    int blk = first + wave;
    Ids next = fetch(blk);
    if (blk < end) load(next);
    next = fetch(blk + NW);

    // q-hat * scale * log2 e: column lr is query head head0 + lr (heads past the group: zeros)
    Split<S> qf[KS];
    {
      const int tr = table_row(p.positions ? p.positions[b] : len - 1 - p.has_cls, p.n_pos);
      const S* qp = static_cast<const S*>(p.q) + b * p.sq[0] + (head0 + (lr < nq ? lr : 0)) * p.sq[1];
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        float x[8], cs[8];
        load8<S>(qp + (32 * s + 8 * lg) * p.sq[2], p.sq[2], p.vec_q, x);
        table_load4(p.cosp, p.sinp, tr, D / 2, 16 * s + 4 * lg, cs);
        rope_rotate8(x, cs);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (lr < nq ? x[e] * p.c2 : 0.f) + 0.f;
        qf[s].set(x);
      }
    }
    f32x4 acc[DT];
    float m_run = -INFINITY, l_run = 0.f, thr = -INFINITY;
    f32x4 nm4 = f32x4{0.f, 0.f, 0.f, 0.f};   // minus the running max (0 before the first row)
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};

    while (blk < end) {
      const unsigned have = rows;
      if (have != 0xffffffffu) {   // uniform: rows that do not exist count as zeros, whatever was read
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bool in = have >> (16 * h + vrow) & 1;
#pragma unroll
          for (int j = 0; j < VJ; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) vr[h][j][e] = in ? vr[h][j][e] : 0u;
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < VJ; ++j)
          *reinterpret_cast<V16*>(vs + T::at(16 * h + vrow, (vch + 4 * j) * T::EPC)) = vr[h][j];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");   // (LDS serves a wave in order)

      f32x4 sacc[2];
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          Frag a;
          __builtin_memcpy(&a, &kr[h][s], sizeof(a));
          sacc[h] = qf[s].mma(a, s == 0 ? nm4 : sacc[h]);
        }
      blk += NW;
      if (blk < end) load(next);
      next = fetch(blk + NW);

      if (have != 0xffffffffu) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) sacc[h][i] = have >> (16 * h + 4 * lg + i) & 1 ? sacc[h][i] : -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h) mx = fmaxf(mx, fmaxf(fmaxf(sacc[h][0], sacc[h][1]), fmaxf(sacc[h][2], sacc[h][3])));
      if (__any(mx > thr)) {   // (as in the forward over packed sequences)
        thr = kSeqSlack + kWeightUp<S>;
        const float old = m_run == -INFINITY ? 0.f : m_run;
        const float mnew = fmaxf(m_run, group4_max(mx) + old - kWeightUp<S>);
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
      for (int d = 0; d < DT; ++d) acc[d] = pf.mma(frag.col(vs, d), acc[d]);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
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
    const float mine = m_run == -INFINITY ? 0.f : fast_exp2(m_run - m);
    float* const out = sums + wave * WS + lr * D;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const f32x4 x = acc[d] * mine;
      *reinterpret_cast<f32x4*>(out + 16 * d + 4 * lg) = x;
    }
    lds_barrier();
    const bool whole = first == 0 && end == blocks;   // the sequence is this worker's alone
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
      if (whole) {
        const float inv = lq > 0.f ? 1.f / lq : 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= inv;
        put_row8<S>(static_cast<S*>(p.o) + ((int64_t)b * p.H + head0 + q) * D + c, x);
      } else {   // (worker, sequence) pairs number worker + sequence: each step is to the next of one
        const int64_t row = (int64_t)(worker + b) * p.H + head0 + q;
        put_row8<float>(p.sums + row * D + c, x);
        if (c == 0) {
          p.stats[row * 2] = mq;
          p.stats[row * 2 + 1] = lq;
        }
      }
    }
    if (p.direct) return;
    // the join's: the sequence's first worker, and how many have a part of it
    if (first == 0 && tid == 0 && hx == 0) {
      p.owners[2 * b] = worker;
      p.owners[2 * b + 1] = blocks ? (int)((before + blocks - 1) / size) - worker + 1 : 0;
    }
    at += end - first;
    if (at >= stop) return;
    before += blocks;
    first = 0;
    do {   // (blocks are left, so a sequence with rows follows)
      if (++b == p.B) return;
    } while (cached_rows(p, b) == 0);
    lds_barrier();   // the sums have been read
  }
}

// O of the sequences that more than one worker had a part of, and zeros of those without
// rows.  A workgroup takes one sequence and query head: its D / 4 channel quads times
// groups of the workers, whose sums are then added.
template <typename S, int D>
__global__ void __launch_bounds__(256) decode_join_kernel(const DecodeParams p) {
  constexpr int Q = D / 4, GR = 256 / Q;
  __shared__ float sums[GR][D];
  __shared__ float sl[GR];
  const int tid = thread_id(), lane = tid & 63;
  const int b = block_id() / p.H, h = block_id() % p.H;
  const int blocks = cached_blocks(p, b);
  S* const o = static_cast<S*>(p.o) + ((int64_t)b * p.H + h) * D;
  if (blocks == 0) {
    if (tid < D / 8) {
      const float z[8] = {};
      put_row8<S>(o + 8 * tid, z);
    }
    return;
  }
  const int w0 = p.owners[2 * b], n = p.owners[2 * b + 1];
  if (n <= 1) return;   // (finished by its worker)
  const int64_t row0 = (int64_t)(w0 + b) * p.H + h;
  float m = -INFINITY;
  for (int i = lane; i < n; i += 64) m = fmaxf(m, p.stats[(row0 + (int64_t)i * p.H) * 2]);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) m = fmaxf(m, __int_as_float(__builtin_amdgcn_ds_bpermute(4 * (lane ^ d), __float_as_int(m))));
  const int g = tid / Q, c = 4 * (tid % Q);
  float l = 0.f;
  f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int i = g; i < n; i += GR) {
    const int64_t row = row0 + (int64_t)i * p.H;
    const float mi = p.stats[row * 2], a = mi == -INFINITY ? 0.f : fast_exp2(mi - m);
    l += a * p.stats[row * 2 + 1];
    x += a * *reinterpret_cast<const f32x4*>(p.sums + row * D + c);
  }
  *reinterpret_cast<f32x4*>(&sums[g][c]) = x;
  if (c == 0) sl[g] = l;
  lds_barrier();
  if (g) return;
#pragma unroll
  for (int i = 1; i < GR; ++i) {
    x += *reinterpret_cast<const f32x4*>(&sums[i][c]);
    l += sl[i];
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  const float y[4] = {x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv};
  store4<S>(o + c, 1, true, y);
}

template <typename S, int D>
static hipError_t decode(const DecodeParams& p, hipStream_t st) {
  hipLaunchKernelGGL((decode_kernel<S, D>), dim3((unsigned)(p.Hkv * p.g_tiles) * (unsigned)p.workers), dim3(64 * kDecodeNW), 0, st, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.direct) return e;
  hipLaunchKernelGGL((decode_join_kernel<S, D>), dim3((unsigned)p.B * p.H), dim3(256), 0, st, p);
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
