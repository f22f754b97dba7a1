// Rows and pages of a paged cache, after they have been written: the rows of
// accepted drafted tokens move up, and places of a batch continue others'
// sequences, sharing, copying, reserving and freeing pages.
//
// Both are copies of whole rows and bound by memory, small calls by the round
// trips of their page numbers and by the launches.  Measured (us a call): accepted tokens of one tree of 8, 12 heads, D 64
// 5.7, of 128 trees of 64, 8 heads, D 128 7.7; 4 places of one prompt forked 9 to 10, 256 places, 8 a prompt, pages of 128
// rows, 8 heads, D 128, fp16 26 to 27 (122 MB read and written, 4.6 TB/s with both launches).
#include "seq.h"

namespace farope {

// Row `pos` of sequence b in a cache with strides st, in elements; -1: not in the cache.
__device__ __forceinline__ int64_t cache_row(const CacheParams& c, const int64_t (&st)[3], int b, int64_t pos) {
  const int64_t place = pos / c.page;
  if (place >= c.max_pages) return -1;
  const int g = c.pages[b * c.spages + place];
  return g < 0 || g >= c.n_pages ? -1 : g * st[0] + (pos - place * c.page) * st[1];
}

// ---------------------------------------------------------------------------
// Row n + i of sequence b becomes what row n + path[b][i] was, for the leading entries
// of path[b] that are 0 or more.  A workgroup takes `1 << lc` 16-byte chunks of all these
// rows of one sequence and cache, kAcceptRows of them a thread: every row is read before
// one is written, so any order of rows, and the same row twice, are right.
// ---------------------------------------------------------------------------
constexpr int kAcceptRows = 8;

__global__ void __launch_bounds__(256) cache_accept_kernel(const AcceptParams p, int lc, int n_grp) {
  const int tid = thread_id(), lane = tid & 63;
  const int b = block_id() / (2 * n_grp), rest = block_id() % (2 * n_grp);
  const bool values = rest >= n_grp;
  const int grp = values ? rest - n_grp : rest;
  const int* const path = p.path + b * p.spath;
  const int n = p.c.lengths[b];
  int count = 0;   // accepted tokens
  for (int i = 0; i < p.cols; i += 64) {
    const int x = i + lane < p.cols ? path[i + lane] : -1;
    const uint64_t end = __builtin_amdgcn_ballot_w64(x < 0);
    count += end ? __builtin_ctzll(end) : 64;
    if (end) break;
  }
  if (rest == 0 && tid == 0) p.out[b] = n < 0 ? n : n > INT32_MAX - count ? INT32_MAX : n + count;
  if (n < 0) return;
  const int64_t(&st)[3] = values ? p.c.svc : p.c.skc;
  char* const base = static_cast<char*>(values ? p.c.vc : p.c.kc);
  const int chunk = (grp << lc) + (tid & ((1 << lc) - 1)), head = chunk / p.cpr;
  const int64_t col = head * st[2] * p.es + (int64_t)(chunk - head * p.cpr) * 16;
  const bool on = head < p.Hkv;
  u32x4 x[kAcceptRows];
  int64_t to[kAcceptRows];
#pragma unroll
  for (int k = 0; k < kAcceptRows; ++k) {
    const int i = (tid >> lc) + k * (256 >> lc);
    to[k] = -1;
    if (on && i < count) {
      const int j = path[i];
      if (j != i) {
        const int64_t from = cache_row(p.c, st, b, (int64_t)n + j);
        to[k] = from < 0 ? -1 : cache_row(p.c, st, b, (int64_t)n + i);
        if (to[k] >= 0) x[k] = *reinterpret_cast<const u32x4*>(base + from * p.es + col);
      }
    }
  }
  // every wave's loads have returned before a store leaves (the compiler moves none past the fence)
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0)
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kAcceptRows; ++k)
    if (to[k] >= 0) *reinterpret_cast<u32x4*>(base + to[k] * p.es + col) = x[k];
}

hipError_t launch_cache_accept(const AcceptParams& p, hipStream_t st) {
  int lc = 8;   // chunks a workgroup takes: so many that its threads hold all rows
  while (lc > 0 && (int64_t)p.cols << lc > 256 * kAcceptRows) --lc;
  const int chunks = p.Hkv * p.cpr, n_grp = (chunks + (1 << lc) - 1) >> lc;
  hipLaunchKernelGGL(cache_accept_kernel, dim3((unsigned)p.B * 2 * n_grp), dim3(256), 0, st, p, lc, n_grp);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Places continue others' sequences, in two launches: the first reads the page tables, lengths
// and reference counts and leaves in the workspace what becomes of them (new table rows with
// the entries that want a page marked, the free pages as bits); the second gives out pages,
// writes, counts and copies.  A page is free if its count was 0 before the call: nothing
// that the call still reads is given out.
// ---------------------------------------------------------------------------
constexpr int kWanted = -2;          // an entry that wants a page

__device__ __forceinline__ int wave_sum(int x) {
  return __builtin_amdgcn_readlane((int)wave_scan((unsigned)x), 63);
}
// Sum over the workgroup's 256 threads.
__device__ __forceinline__ int block_sum(int x, int* share, int tid) {
  x = wave_sum(x);
  __syncthreads();
  if ((tid & 63) == 0) share[tid >> 6] = x;
  __syncthreads();
  return share[0] + share[1] + share[2] + share[3];
}

__global__ void __launch_bounds__(256) cache_plan_kernel(const ForkParams p) {
  __shared__ int share[4];
  const int tid = thread_id(), lane = tid & 63;
  if (block_id() >= p.B) {   // a chunk's free pages
    const int chunk = block_id() - p.B;
    int n = 0;
#pragma unroll
    for (int k = 0; k < kForkChunk / 256; ++k) {
      const int g = chunk * kForkChunk + k * 256 + tid;
      const uint64_t free = __builtin_amdgcn_ballot_w64(g < p.c.n_pages && p.refs[g < p.c.n_pages ? g : 0] == 0);
      n += __builtin_popcountll(free);
      if (lane == 0) p.bits[g >> 6] = free;
    }
    n = block_sum(lane == 0 ? n : 0, share, tid);
    if (tid == 0) p.free[chunk] = n;
    return;
  }
  const int b = block_id(), parent = p.parents[b], M = p.c.max_pages;
  const bool alive = parent >= 0 && parent < p.B;
  const int from = alive ? parent : 0;
  const int64_t most = (int64_t)M * p.c.page;
  const int len = p.c.lengths[from], cut = len < 0 ? 0 : len > most ? (int)most : len;
  const int n = alive ? cut : 0, full = n / p.c.page;
  const int more = alive && p.room ? p.room[b] : 0;
  const int64_t want = ((int64_t)n + (more > 0 ? more : 0) + p.c.page - 1) / p.c.page;
  const int need = alive ? (int)(want < M ? want : M) : 0;
  bool twin = false;   // a place before has the same parent
  for (int i = tid; i < b; i += 256) twin |= p.parents[i] == parent;
  twin = block_sum(twin, share, tid) != 0;
  int wanted = 0;
  for (int i = tid; i < M; i += 256) {
    int g = alive ? p.c.pages[from * p.c.spages + i] : -1, e = -1;
    if (g < 0 || g >= p.c.n_pages) g = -1;
    if (i < full) e = g;
    else if (g >= 0 && !twin && p.refs[g] == 1) e = g;
    else if (i < need) e = kWanted;
    p.table[(int64_t)b * M + i] = e;
    wanted += e == kWanted;
    if (i == full) p.from[b] = e == kWanted && n > full * p.c.page ? g : -1;   // the page whose rows are copied
  }
  wanted = block_sum(wanted, share, tid);
  if (tid == 0) {
    p.wanted[b] = wanted;
    p.len[b] = n;
    if (full >= M) p.from[b] = -1;
  }
}

// The chunk that holds free page number `rank`, and the free pages before it; all 64 lanes
// search together.  n_chunks: there is none.
__device__ __forceinline__ int find_chunk(const ForkParams& p, int rank, int lane, int& before) {
  before = 0;
  for (int i = 0; i < p.chunks; i += 64) {
    const int n = i + lane < p.chunks ? p.free[i + lane] : 0;
    const int sum = (int)wave_scan((unsigned)n);
    const uint64_t past = __builtin_amdgcn_ballot_w64(before + sum > rank);
    if (past) {
      const int l = __builtin_ctzll(past);
      before += __builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(n, l);
      return i + l;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  return p.chunks;
}
// Free page number `rank`; -1: there are not so many.
__device__ __forceinline__ int find_free(const ForkParams& p, int rank, int lane) {
  int before;
  const int chunk = find_chunk(p, rank, lane, before);
  if (chunk == p.chunks) return -1;
  const uint64_t w = lane < kForkChunk / 64 ? p.bits[chunk * (kForkChunk / 64) + lane] : 0;
  const int n = __builtin_popcountll(w), sum = (int)wave_scan((unsigned)n), k = rank - before;
  const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(sum > k));
  int left = k - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(n, l));
  uint64_t bits = (uint64_t)(unsigned)__builtin_amdgcn_readlane((int)(w >> 32), l) << 32 | (unsigned)__builtin_amdgcn_readlane((int)w, l);
  for (; left > 0; --left) bits &= bits - 1;
  return chunk * kForkChunk + 64 * l + __builtin_ctzll(bits);
}

// 16-byte chunks a thread copies.  Each workgroup finds its place's page by itself, a chain of dependent
// reads, so few workgroups with much to copy are better: 8 chunks take 35 us for the 256 places above, 16 take 26 to 27
// (the 4 places: no difference).
constexpr int kCopyChunks = 16;

__global__ void __launch_bounds__(256) cache_fork_kernel(const ForkParams p, int copies) {
  __shared__ int share[4];
  const int tid = thread_id(), lane = tid & 63;
  // places' tables first: `copies` more workgroups a place then copy its rows
  const bool tables = block_id() < p.B;
  const int b = tables ? block_id() : (block_id() - p.B) / copies;
  const int src = p.from[b];
  const int n = p.len[b], row_chunks = p.Hkv * p.cpr;
  const int64_t all = (int64_t)(n % p.c.page) * row_chunks;   // 16-byte chunks of one cache to be copied
  const int64_t at = (int64_t)(tables ? 0 : (block_id() - p.B) % copies) * (256 * kCopyChunks) + tid;
  if (!tables && (src < 0 || at - tid >= 2 * all)) return;
  int first = 0;   // pages that the places before want
  for (int i = tid; i < b; i += 256) first += p.wanted[i];
  first = block_sum(first, share, tid);

  if (!tables) {
    const int dst = find_free(p, first, lane);   // (entry `full` is the first that wants one)
    if (dst < 0) return;
    u32x4 x[kCopyChunks];
    int64_t to[kCopyChunks];
#pragma unroll
    for (int k = 0; k < kCopyChunks; ++k) {
      const int64_t i = at + 256 * k;
      to[k] = -1;
      if (i >= 2 * all) continue;
      const bool values = i >= all;
      const int j = (int)(values ? i - all : i), r = j / row_chunks, c = j - r * row_chunks, head = c / p.cpr;
      const int64_t(&st)[3] = values ? p.c.svc : p.c.skc;
      const int64_t in = (r * st[1] + head * st[2]) * p.es + (int64_t)(c - head * p.cpr) * 16;
      to[k] = dst * st[0] * p.es + in;
      x[k] = *reinterpret_cast<const u32x4*>(static_cast<const char*>(values ? p.c.vc : p.c.kc) + src * st[0] * p.es + in);
    }
#pragma unroll
    for (int k = 0; k < kCopyChunks; ++k)
      if (at + 256 * k < 2 * all) *reinterpret_cast<u32x4*>(static_cast<char*>(at + 256 * k >= all ? p.c.vc : p.c.kc) + to[k]) = x[k];
    return;
  }

  const int wanted = p.wanted[b], M = p.c.max_pages;
  if (b == p.B - 1) {   // pages that are wanted and not there
    int n = 0;
    for (int i = tid; i < p.chunks; i += 256) n += p.free[i];
    n = block_sum(n, share, tid);
    if (tid == 0) p.missing[0] = first + wanted > n ? first + wanted - n : 0;
  }
  // the place's pages, in ascending order, to its part of the list
  if (wanted) {
    int before;
    for (int chunk = find_chunk(p, first, lane, before); chunk < p.chunks && before < first + wanted; ++chunk) {
      const uint64_t w = lane < kForkChunk / 64 ? p.bits[chunk * (kForkChunk / 64) + lane] : 0;
      int at = before + (int)wave_scan((unsigned)__builtin_popcountll(w)) - __builtin_popcountll(w);
      if (tid < 64)
        for (uint64_t left = w; left; left &= left - 1, ++at)
          if (at >= first && at < first + wanted) p.list[at] = chunk * kForkChunk + 64 * lane + __builtin_ctzll(left);
      before += p.free[chunk];
    }
    // (`before` is now the free pages up to the place's last, or all of them)
    const int got = before < first + wanted ? before - first : wanted;
    __syncthreads();
    int done = 0;   // entries served
    for (int i0 = 0; i0 < M; i0 += 256) {
      const int i = i0 + tid, e = i < M ? p.table[(int64_t)b * M + i] : -1;
      const uint64_t m = __builtin_amdgcn_ballot_w64(e == kWanted);
      __syncthreads();
      if (lane == 0) share[tid >> 6] = __builtin_popcountll(m);
      __syncthreads();
      int k = done + __builtin_amdgcn_mbcnt_hi((unsigned)(m >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)m, 0u));
      for (int w = 0; w < tid >> 6; ++w) k += share[w];
      if (e == kWanted) p.table[(int64_t)b * M + i] = k < got ? p.list[first + k] : -1;
      done += share[0] + share[1] + share[2] + share[3];
    }
  }
  // (each thread reads the entries that it wrote)
  for (int i = tid; i < M; i += 256) {
    int* const at = p.pages + b * p.c.spages + i;
    const int old = *at, now = p.table[(int64_t)b * M + i];
    if (old != now) {
      if (old >= 0 && old < p.c.n_pages) atomicAdd(p.refs + old, -1);
      if (now >= 0) atomicAdd(p.refs + now, 1);
      *at = now;
    }
  }
  if (tid == 0) p.lengths[b] = p.len[b];
}

hipError_t launch_cache_fork(const ForkParams& p, hipStream_t st) {
  const int64_t chunks = 2 * (int64_t)p.c.page * p.Hkv * p.cpr, per = 256 * kCopyChunks;
  const int copies = (int)((chunks + per - 1) / per);
  hipLaunchKernelGGL(cache_plan_kernel, dim3((unsigned)p.B + p.chunks), dim3(256), 0, st, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(cache_fork_kernel, dim3((unsigned)p.B * (1 + copies)), dim3(256), 0, st, p, copies);
  return hipGetLastError();
}

}  // namespace farope
