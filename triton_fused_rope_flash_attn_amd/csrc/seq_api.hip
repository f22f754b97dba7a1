// C-ABI layer of attention over packed sequences and over a paged cache:
// argument checks, workspaces and dispatch.  Declarations: include/farope.h.
#include "farope.h"

#include "params.h"
#include "seq_params.h"

using namespace farope;

namespace {

int elem_size(int dt) { return dt == FAROPE_F32 ? 4 : 2; }

int check_desc(const farope_seq_desc* d, bool queries) {
  if (!d) return FAROPE_ERR_NULL;
  if (d->tokens < 0 || d->seqs < 1 || d->kv_heads < 1) return FAROPE_ERR_SHAPE;
  if (queries && (d->heads < 1 || d->heads % d->kv_heads)) return FAROPE_ERR_SHAPE;
  if (d->head_dim != 32 && d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256) return FAROPE_ERR_HEAD_DIM;
  if (d->dtype != FAROPE_F32 && d->dtype != FAROPE_F16 && d->dtype != FAROPE_BF16) return FAROPE_ERR_DTYPE;
  if (d->n_pos < 1) return FAROPE_ERR_TABLE;
  if (d->has_cls != 0 && d->has_cls != 1) return FAROPE_ERR_SEQ_LEN;
  return FAROPE_OK;
}
int check_ptr(const void* p, int align) {
  if (!p) return FAROPE_ERR_NULL;
  return reinterpret_cast<uintptr_t>(p) % align ? FAROPE_ERR_ALIGN : FAROPE_OK;
}
#define FAROPE_TRY(expr)                \
  do {                                  \
    const int rc__ = (expr);            \
    if (rc__ != FAROPE_OK) return rc__; \
  } while (0)
int launch_rc(hipError_t e) { return e == hipSuccess ? FAROPE_OK : FAROPE_ERR_LAUNCH; }

// 16-byte access to 8 channels of any row
int vec_rows(const void* p, const int64_t s[3], int es) {
  return s[2] == 1 && reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[0] * es % 16 == 0 && s[1] * es % 16 == 0;
}
// ... and rows that a stage's loads reach by 32-bit offsets from a sequence's first row.
// The offsets run up to kPad rows past a sequence's end and must not wrap.
constexpr int64_t kPad = 256;
bool offsets_fit(int64_t tokens, int64_t row_bytes) { return row_bytes < (int64_t(1) << 31) / (tokens + kPad); }
bool streams(const farope_seq_desc* d, const void* p, const int64_t s[3]) {
  const int es = elem_size(d->dtype);
  return vec_rows(p, s, es) && s[0] >= 0 && s[0] < (int64_t(1) << 31) && offsets_fit(d->tokens, s[0] * es);
}

// Workgroups of the kernels that take 2048 / head_dim tokens and four key heads each.
int64_t token_blocks(const farope_seq_desc* d) {
  const int64_t per = 2048 / d->head_dim;
  return (d->tokens + per - 1) / per * (((int64_t)d->kv_heads + 3) / 4);
}

// Sizes that the kernels' 32-bit offsets and the launches hold.
int check_sizes(const farope_seq_desc* d) {
  const int64_t row = (int64_t)d->head_dim * elem_size(d->dtype), T = d->tokens;
  if (!offsets_fit(T, row)) return FAROPE_ERR_SHAPE;               // rows of the workspace
  if (d->heads * row > (int64_t(1) << 24)) return FAROPE_ERR_SHAPE;   // (a tile's rows of an output)
  if (seq_slots(d->tokens, d->seqs, 6) * d->heads > kMaxWorkgroups) return FAROPE_ERR_SHAPE;
  // (with the workgroups that find the slots' tiles)
  return token_blocks(d) + seq_slots(d->tokens, d->seqs, 6) > kMaxWorkgroups ? FAROPE_ERR_SHAPE : FAROPE_OK;
}

// Workgroups of a call over a paged cache that are resident at once (decode_kernel's registers):
// one round of workers, whose shares are equal, is the fastest, so never more than these (a few more
// start a whole share on an idle chip: 516 / 504 for 12 key heads, D 128, 2 x 32768 97 / 83; 264 / 252 at D
// 256, 8 x 8192 209 / 156).  Measured (us, 512 / 768 / 1024
// workgroups; "sequences x rows, key heads"), D 128: 1 x 32768, 8 37.5 / 43.4 / 46.0, 32 x 8192, 1
// 35.5 / 44.6 / 41.5; D 64: 16 x 2048, 12 30.8 / 27.1 / 32.6; D 256, 256 / 512: 8 x 8192, 2 40 / 53.
int64_t decode_wgs(const farope_seq_desc* d) {
  const int row = d->head_dim * elem_size(d->dtype);
  return (int64_t)kCus * (row <= 64 ? 4 : row == 128 ? 3 : row == 256 ? 2 : 1);
}

// Token i sees j <= i with i - j < window or j < sinks; window 0: as the descriptor says.
struct Window {
  int32_t window, sinks;
};
// A window that holds every row that a sequence can have is none.
Window window_of(const farope_seq_desc* d, int32_t window, int32_t sinks) {
  if (window >= d->tokens) return Window{0, 0};
  return Window{window, sinks < d->tokens ? sinks : d->tokens};
}
farope_seq_desc causal_desc(const farope_seq_desc* d) {
  farope_seq_desc c = *d;
  c.causal = 1;
  return c;
}

// Workspace, in fp32 elements, each part from a 256-byte boundary.
constexpr int kMaxParts = 8;
struct SeqWs {
  int64_t khat, vcopy, map_q, map_k, qhat, gcopy, nl, nd, ng, pk, pv, spk, spv, total;
};
// Parts that the queries of a key tile (64 rows) are divided into, joined by a launch of its
// own: so many that about four workgroups per CU share the work, but none below a stage of
// queries on average.  Measured (us, forward and backward, 1 / 2 / 4 parts; workgroups of
// one part in brackets), D 128: 16384 tokens, 2 key heads [514] 3837 / 2839 / 2832, 4096, 4
// [264] 713 / 523 / 432, 1024, 4 [72] 181 / 129 / 105, 8 x 1024, 8 [1096] 208 / 239 / 311; D 64:
// 2048, 2 [68] 204 / 138 / 105, 4 x 2048, 8 [1064] 180 / 179 / 196; D 256: 2 x 4096, 8 [1048] 1251 /
// 1347 / 1525; fp32, D 64: 3 up to 257, 4 [44] 100 / 79 / 72.
// With a window key tiles have like work, so the chip should end its last round of workgroups full: the parts with the
// fewest stages one after the other, a part's sums, written and read, counted in stages too (at 4.9 TB/s, of 2.7 us).
// Measured (us, forward and backward, 1 / 2 / 3 / 4 parts), D 128: 16384 tokens, 2 key heads, window 1024 450 / 475 / 498 / 506; fp32, D 64: 3 up
// to 513, 4, window 100 149 / 105 / 90 / 86.
int64_t dkdv_resident(const farope_seq_desc* d) {   // workgroups of seq_dkdv_kernel, by its registers and LDS
  const int row = d->head_dim * elem_size(d->dtype);
  return (int64_t)kCus * (d->dtype == FAROPE_F32 ? row <= 256 ? 2 : 1 : row <= 128 ? 4 : row == 256 ? 2 : 1);
}
int64_t window_stages(const farope_seq_desc* d, Window win) {
  const int64_t mean = d->tokens / d->seqs;
  return (int64_t)(d->heads / d->kv_heads) * ((mean < win.window ? mean : win.window) / 64 + 2);
}
// Parts of the key tiles' queries that the launches of seq_dkdv_kernel and seq_join_kernel hold.
bool parts_fit(const farope_seq_desc* d, int64_t parts) {
  return seq_slots(d->tokens, d->seqs, 6) * d->kv_heads * parts <= kMaxWorkgroups &&
         ((int64_t)d->tokens * d->head_dim / 2048 + 1) * d->kv_heads <= kMaxWorkgroups;
}
int window_parts(const farope_seq_desc* d, Window win) {
  // (tiles, not slots: a sequence ends half a tile before its last one's end)
  const int64_t wgs = (d->tokens / 64 + (d->seqs + 1) / 2 * (d->seqs > 1)) * d->kv_heads, slots = dkdv_resident(d), stages = window_stages(d, win);
  const double sums = (double)d->tokens * d->kv_heads * d->head_dim * 1.2e-6;
  int best = 1;
  double least = 0;
  for (int parts = 1; parts <= kMaxParts && parts <= stages; ++parts) {
    if (parts > 1 && !parts_fit(d, parts)) break;
    const int64_t rounds = (wgs * parts + slots - 1) / slots;
    const double cost = (double)stages * (rounds < 1 ? 1 : rounds) / parts + (parts > 1 ? parts * sums : 0.);
    if (parts == 1 || cost < least) {
      best = parts;
      least = cost;
    }
  }
  return best;
}
int dkdv_parts(const farope_seq_desc* d, Window win) {
  const int64_t wgs = seq_slots(d->tokens, d->seqs, 6) * d->kv_heads;
  if (win.window) return window_parts(d, win);
  const int64_t stages = (int64_t)(d->heads / d->kv_heads) * (d->tokens / d->seqs / 64 + 1);
  int64_t parts = (4 * kCus + wgs / 2) / wgs;
  if (parts > kMaxParts) parts = kMaxParts;
  if (parts > stages) parts = stages;
  return parts < 1 ? 1 : (int)parts;
}
// Short sequences: the tile kernels rotate K themselves.  Measured (us, rotated rows in a pass of
// their own / rotated by the tiles; "sequences x tokens, heads", B backward too), D 64: 1 x 197, 12
// 13.5 / 9.0, 4 x 197, 12 11.2 / 9.0, B 58 / 49, 64 x 100, 12 25.2 / 20.1, B 79 / 75, 1 x 400, 12 11.5 /
// 12.4, 64 x 150, 12 B 103 / 104, 64 x 197, 12 36.0 / 36.8, 1 x 1024, 16 16 / 23; D 32: 128 up to 100, 8
// B 91 / 81; D 128: 1 x 100, 8 11.4 / 9.4, 1 x 197, 12 13.0 / 13.3, 4 x 512, 16 23 / 28.
// All of these are of like lengths.  The host knows the mean alone, which does not show one long sequence
// beside many short ones: 8192 tokens and 100 of 1 to 30 (mean 96), 8 heads, D 64 take 224 us, B 688, where the
// long one alone takes 100, B 428.
bool rotates_itself(const farope_seq_desc* d, bool v_streams) {
  if (!v_streams || d->head_dim > 128) return false;
  const int mean = d->tokens / d->seqs;
  if (d->head_dim == 128) return d->tokens <= 128;
  return mean <= 128 || (mean <= 256 && d->tokens <= 1024);
}
// Key tiles with sinks, which every later query sees: where that is more than half as much again as other tiles have,
// parts of their queries of 8 stages, or of a workgroup's for other tiles where these are fewer (0: they are not
// divided).  Measured (us, forward and backward of 16384 tokens, 8 heads, 2 of keys, D 128, window 1024, 4 sinks):
// parts as large as the other workgroups' and at the launch's front 504, of 16 stages and at its end 473, of 8 450.  Undivided / divided,
// the sinks' tile having r times the others' stages: 8 x 2048, 32 heads, 8 of keys, D 128, window 512 [r 3.3] 1157 / 1017, 1024 [1.8]
// 1392 / 1301, 1300 [1.5] 1512 / 1515, 1536 [1.3] 1550 / 1576; 2 x 4096, 16, 4 of keys, D 64, 1024 [3.6] 307 / 263, 2048 [1.9] 335 / 338, 3000
// [1.3] 396 / 405; one of 16384, 8, 2 of keys, D 128, few workgroups, 12000 [1.4] 3220 / 2657.
// No more parts than one resident round of workgroups: many tiles fill the chip by themselves, and each part has its sums,
// 2 * 64 * D in fp32, in the workspace, 32 MB of them at most.  Measured (us, one round / two / four / no such bound; 32 heads, 8 of
// keys, D 128): 16384 tokens, window 1024, 4 sinks 1557 / 1554 / 1555 / 1551, 1024 2501 / 2535 / 2588 / 3070, 4096 4970 / 5026 /
// 5096 / 7575; 32 x 4096, window 512, 256 sinks 9416 / 9470 / 9211 / 10230, 2048 18200 / 18200 / 18240 / 28000; 64 x 1024, 8 heads, D 64,
// window 64, 4 sinks 473 / 481 / 491 / 492.
constexpr int kMaxSinkParts = 128;
int sink_tiles(Window win) { return win.window ? (int)(((int64_t)win.sinks + 63) / 64) : 0; }
int sink_parts(const farope_seq_desc* d, Window win) {
  if (!sink_tiles(win)) return 0;
  const int64_t all = (int64_t)(d->heads / d->kv_heads) * (d->tokens / d->seqs / 64 + 1);
  if (2 * all <= 3 * window_stages(d, win)) return 0;
  int64_t part = window_stages(d, win) / window_parts(d, win);
  part = part > 8 ? 8 : part < 1 ? 1 : part;
  int64_t n = (all + part - 1) / part;
  if (n > kMaxSinkParts) n = kMaxSinkParts;
  const int64_t tiles = (int64_t)d->seqs * sink_tiles(win) * d->kv_heads;
  if (n > dkdv_resident(d) / tiles) n = dkdv_resident(d) / tiles;
  // (and none where the launch does not hold them; sink_join_kernel has 64 workgroups a tile, of which there are few here)
  const int64_t others = seq_slots(d->tokens, d->seqs, 6) * d->kv_heads * window_parts(d, win);
  return n < 2 || others + tiles * n > kMaxWorkgroups ? 0 : (int)n;
}
int64_t sink_workgroups(const farope_seq_desc* d, Window win) {
  return (int64_t)d->seqs * sink_tiles(win) * sink_parts(d, win) * d->kv_heads;
}
SeqWs seq_ws(const farope_seq_desc* d, bool backward, bool v_streams, bool g_streams, Window win) {
  const int64_t es = elem_size(d->dtype), kv = (int64_t)d->tokens * d->kv_heads * d->head_dim * es / 4;
  const int64_t q = (int64_t)d->tokens * d->heads * d->head_dim * es / 4, rows = (int64_t)d->tokens * d->heads;
  auto al = [](int64_t x) { return (x + 63) & ~int64_t(63); };
  SeqWs w{};
  const bool pass = !rotates_itself(d, v_streams);
  const int64_t slots = pass ? al(4 * seq_slots(d->tokens, d->seqs, 6)) : 0;
  w.vcopy = pass ? al(kv) : 0;
  w.map_q = w.vcopy + (v_streams ? 0 : al(kv));
  w.map_k = w.map_q + slots;
  w.qhat = w.map_k + (backward ? slots : 0);
  w.gcopy = w.qhat + (backward ? al(q) : 0);
  w.nl = w.gcopy + (backward && !g_streams ? al(q) : 0);
  w.nd = w.nl + (backward ? al(rows) : 0);
  const int parts = backward ? dkdv_parts(d, win) : 1;
  const int64_t sums = parts > 1 ? al((int64_t)parts * d->tokens * d->kv_heads * d->head_dim) : 0;
  w.ng = w.nd + (backward ? al(rows) : 0);
  w.pk = w.ng + (backward && d->dtype == FAROPE_F16 && d->head_dim == 128 ? al(rows) : 0);
  w.pv = w.pk + sums;
  w.spk = w.pv + sums;
  const int64_t sink_sums = backward ? al(sink_workgroups(d, win) * 64 * d->head_dim) : 0;
  w.spv = w.spk + sink_sums;
  w.total = w.spv + sink_sums;
  return w;
}

void place(SeqParams& p, const farope_seq_desc* d, const SeqWs& w, float* ws, bool backward, bool v_streams, bool g_streams,
           Window win) {
  p.window = win.window;
  p.sinks = win.sinks;
  if (!rotates_itself(d, v_streams)) {
    p.khat = ws;
    p.map_q = reinterpret_cast<int*>(ws + w.map_q);
    if (backward) p.map_k = reinterpret_cast<int*>(ws + w.map_k);
  }
  if (!v_streams) p.vcopy = ws + w.vcopy;
  if (!backward) return;
  p.qhat = ws + w.qhat;
  if (!g_streams) p.gcopy = ws + w.gcopy;
  p.nl = ws + w.nl;
  p.nd = ws + w.nd;
  p.ng = ws + w.ng;
  p.pk = ws + w.pk;
  p.pv = ws + w.pv;
  p.parts = dkdv_parts(d, win);
  p.spk = ws + w.spk;
  p.spv = ws + w.spv;
  p.sink_tiles = sink_tiles(win);
  p.sink_parts = sink_parts(d, win);
}

void fill(SeqParams& p, const farope_seq_desc* d, const void* q, const int64_t sq[3], const void* k, const int64_t sk[3],
          const void* v, const int64_t sv[3], const float* cosp, const float* sinp, const int32_t* positions,
          const int32_t* cu) {
  const int es = elem_size(d->dtype);
  p.q = q; p.k = k; p.v = v;
  for (int i = 0; i < 3; ++i) { p.sq[i] = sq[i]; p.sk[i] = sk[i]; p.sv[i] = sv[i]; }
  p.vec_q = vec_rows(q, sq, es); p.vec_k = vec_rows(k, sk, es); p.vec_v = vec_rows(v, sv, es);
  p.cosp = cosp; p.sinp = sinp; p.positions = positions; p.cu = cu;
  p.T = d->tokens; p.B = d->seqs; p.H = d->heads; p.Hkv = d->kv_heads;
  p.n_pos = d->n_pos; p.has_cls = d->has_cls; p.causal = d->causal != 0;
  p.scale = d->softmax_scale;
  p.c2 = d->softmax_scale * 1.4426950408889634f;
}

int check_inputs(const farope_seq_desc* d, const void* q, const int64_t* sq, const void* k, const int64_t* sk, const void* v,
                 const int64_t* sv, const float* cosp, const float* sinp, const int32_t* positions, const int32_t* cu) {
  FAROPE_TRY(check_desc(d, true));
  if (!sq || !sk || !sv) return FAROPE_ERR_NULL;
  FAROPE_TRY(check_sizes(d));
  const int es = elem_size(d->dtype);
  FAROPE_TRY(check_ptr(q, es));
  FAROPE_TRY(check_ptr(k, es));
  FAROPE_TRY(check_ptr(v, es));
  FAROPE_TRY(check_ptr(cosp, 16));
  FAROPE_TRY(check_ptr(sinp, 16));
  if (positions) FAROPE_TRY(check_ptr(positions, 4));
  return check_ptr(cu, 4);
}

int seq_fwd_call(const farope_seq_desc* desc, Window win, const void* q, const int64_t q_stride[3], const void* k,
                   const int64_t k_stride[3], const void* v, const int64_t v_stride[3], const float* cosp, const float* sinp,
                   const int32_t* positions, const int32_t* cu, void* o, float* lse, float* ws, size_t ws_elems, void* stream) {
  FAROPE_TRY(check_desc(desc, true));
  if (desc->tokens == 0) return FAROPE_OK;
  FAROPE_TRY(check_inputs(desc, q, q_stride, k, k_stride, v, v_stride, cosp, sinp, positions, cu));
  FAROPE_TRY(check_ptr(o, 16));
  FAROPE_TRY(check_ptr(lse, 4));
  const bool vs = streams(desc, v, v_stride);
  const SeqWs w = seq_ws(desc, false, vs, true, win);
  if (w.total) FAROPE_TRY(check_ptr(ws, 16));
  if ((int64_t)ws_elems < w.total) return FAROPE_ERR_SCRATCH;
  SeqParams p{};
  fill(p, desc, q, q_stride, k, k_stride, v, v_stride, cosp, sinp, positions, cu);
  p.o = o; p.lse = lse;
  place(p, desc, w, ws, false, vs, true, win);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (p.khat) FAROPE_TRY(launch_rc(launch_seq_prep(p, desc->dtype, desc->head_dim, false, st)));
  return launch_rc(launch_seq_fwd(p, desc->dtype, desc->head_dim, st));
}

int seq_bwd_call(const farope_seq_desc* desc, Window win, const void* q, const int64_t q_stride[3], const void* k,
                   const int64_t k_stride[3], const void* v, const int64_t v_stride[3], const void* o, const void* dout,
                   const int64_t dout_stride[3], const float* lse, const float* cosp, const float* sinp,
                   const int32_t* positions, const int32_t* cu, void* dq, void* dk, void* dv, float* ws, size_t ws_elems,
                   void* stream) {
  FAROPE_TRY(check_desc(desc, true));
  if (desc->tokens == 0) return FAROPE_OK;
  FAROPE_TRY(check_inputs(desc, q, q_stride, k, k_stride, v, v_stride, cosp, sinp, positions, cu));
  if (!dout_stride) return FAROPE_ERR_NULL;
  const int es = elem_size(desc->dtype);
  FAROPE_TRY(check_ptr(dout, es));
  FAROPE_TRY(check_ptr(o, 16));
  FAROPE_TRY(check_ptr(lse, 4));
  FAROPE_TRY(check_ptr(dq, 16));
  FAROPE_TRY(check_ptr(dk, 16));
  FAROPE_TRY(check_ptr(dv, 16));
  FAROPE_TRY(check_ptr(ws, 16));
  const bool vs = streams(desc, v, v_stride), gs = streams(desc, dout, dout_stride);
  const SeqWs w = seq_ws(desc, true, vs, gs, win);
  if ((int64_t)ws_elems < w.total) return FAROPE_ERR_SCRATCH;
  SeqParams p{};
  fill(p, desc, q, q_stride, k, k_stride, v, v_stride, cosp, sinp, positions, cu);
  p.dout = dout;
  for (int i = 0; i < 3; ++i) p.sdo[i] = dout_stride[i];
  p.vec_do = vec_rows(dout, dout_stride, es);
  p.o = const_cast<void*>(o);
  p.lse = const_cast<float*>(lse);
  p.dq = dq; p.dk = dk; p.dv = dv;
  place(p, desc, w, ws, true, vs, gs, win);
  return launch_rc(launch_seq_bwd(p, desc->dtype, desc->head_dim, static_cast<hipStream_t>(stream)));
}

int check_cache(const farope_seq_desc* d, const farope_cache_desc* c, const int32_t* table, const int32_t* lengths) {
  if (!c) return FAROPE_ERR_NULL;
  if (c->pages < 1 || c->page_rows < 1 || c->max_pages < 1 || c->table_stride < 0) return FAROPE_ERR_SHAPE;
  FAROPE_TRY(check_ptr(c->k, 16));
  FAROPE_TRY(check_ptr(c->v, 16));
  for (int i = 0; i < 3; ++i)
    if (c->k_stride[i] * elem_size(d->dtype) % 16 || c->v_stride[i] * elem_size(d->dtype) % 16) return FAROPE_ERR_ALIGN;
  FAROPE_TRY(check_ptr(table, 4));
  return check_ptr(lengths, 4);
}
CacheParams cache_params(const farope_cache_desc* c, const int32_t* table, const int32_t* lengths) {
  CacheParams p{};
  p.kc = c->k; p.vc = c->v;
  for (int i = 0; i < 3; ++i) { p.skc[i] = c->k_stride[i]; p.svc[i] = c->v_stride[i]; }
  p.pages = table; p.spages = c->table_stride; p.lengths = lengths;
  p.n_pages = c->pages; p.page = c->page_rows; p.max_pages = c->max_pages;
  return p;
}

// Workers among which a key head's cached rows are divided (decode.hip).  The lengths stay on
// the device, so the rules go by the sequences' number and room.
int decode_tiles(const farope_seq_desc* d) { return (d->heads / d->kv_heads + 15) / 16; }
// One worker per sequence, nothing to join, where a sequence's room is short, or up to 2048
// rows where the sequences alone make several rounds (up to 1024, one).  Measured (us, even
// shares / one per sequence): 1 x 197, 12 heads, D 64 11.1 / 6.9; 256 sequences up to 1024, 8
// heads, D 128 104 / 89; 64 x 1024, 16 heads, D 64 66 / 59; 5 up to 1025, 8 heads, fp32 14.4 / 19.3.
// (So a short sequence in a wide table pays for the join: 197 rows, 12 heads, D 64 7 us with room for 197, 9 for
// 512, 13 for 1024 to 131072.)
// (With a window the rules go by the rows that it leaves.)
int64_t decode_room(const farope_cache_desc* c, int32_t window, int32_t sinks) {
  const int64_t room = (int64_t)c->max_pages * c->page_rows;
  const int64_t rows = window ? ((int64_t)window + 31) / 32 * 32 + 32 + ((int64_t)sinks + 31) / 32 * 32 : room;
  return rows < room ? rows : room;
}
bool decode_direct(const farope_seq_desc* d, const farope_cache_desc* c, int32_t window, int32_t sinks) {
  const int64_t room = decode_room(c, window, sinks), wgs = (int64_t)d->seqs * d->kv_heads * decode_tiles(d);
  return room <= 512 || (room <= 1024 && wgs >= decode_wgs(d)) || (room <= 2048 && wgs >= 2 * decode_wgs(d));
}
int decode_workers(const farope_seq_desc* d, const farope_cache_desc* c, int32_t window, int32_t sinks) {
  if (decode_direct(d, c, window, sinks)) return d->seqs;
  const int64_t heads = (int64_t)d->kv_heads * decode_tiles(d);
  // (a worker has 128 rows at least)
  const int64_t most = d->seqs * ((decode_room(c, window, sinks) + 127) / 128);
  int64_t n = decode_wgs(d) / heads;
  if (n < 1) n = 1;
  return (int)(n < most ? n : most);
}
// Workspace, in fp32 elements, each part from a 16-byte boundary: sums, their statistics, owners.
struct DecodeWs {
  int64_t stats, owners, total;
};
DecodeWs decode_ws(const farope_seq_desc* d, const farope_cache_desc* c, int32_t window, int32_t sinks) {
  if (decode_direct(d, c, window, sinks)) return DecodeWs{};
  const int64_t rows = ((int64_t)decode_workers(d, c, window, sinks) + d->seqs) * d->heads;
  DecodeWs w{};
  w.stats = rows * d->head_dim;
  w.owners = (w.stats + 2 * rows + 3) & ~int64_t(3);
  w.total = w.owners + 2 * (int64_t)d->seqs;
  return w;
}

// A window that holds every row that a sequence can have is none.
int32_t decode_window(const farope_cache_desc* c, int32_t window) {
  return window >= (int64_t)c->max_pages * c->page_rows ? 0 : window;
}
int decode_call(const farope_seq_desc* desc, int32_t window, int32_t sinks, const void* q, const int64_t q_stride[3],
                const float* cosp, const float* sinp, const int32_t* positions, const farope_cache_desc* cache,
                const int32_t* page_table, const int32_t* lengths, void* o, float* ws, size_t ws_elems, void* stream) {
  FAROPE_TRY(check_desc(desc, true));
  if (desc->tokens != desc->seqs) return FAROPE_ERR_SHAPE;
  if (!q_stride) return FAROPE_ERR_NULL;
  const int es = elem_size(desc->dtype);
  FAROPE_TRY(check_ptr(q, es));
  FAROPE_TRY(check_ptr(cosp, 16));
  FAROPE_TRY(check_ptr(sinp, 16));
  if (positions) FAROPE_TRY(check_ptr(positions, 4));
  FAROPE_TRY(check_cache(desc, cache, page_table, lengths));
  FAROPE_TRY(check_ptr(o, 16));
  const DecodeWs w = decode_ws(desc, cache, window, sinks);
  if (w.total) {
    FAROPE_TRY(check_ptr(ws, 16));
    if ((int64_t)ws_elems < w.total) return FAROPE_ERR_SCRATCH;
  }
  const int workers = decode_workers(desc, cache, window, sinks);
  if ((int64_t)desc->kv_heads * decode_tiles(desc) * workers > kMaxWorkgroups || (int64_t)desc->seqs * desc->heads > kMaxWorkgroups)
    return FAROPE_ERR_SHAPE;
  DecodeParams p{};
  p.q = q;
  for (int i = 0; i < 3; ++i) p.sq[i] = q_stride[i];
  p.vec_q = vec_rows(q, q_stride, es);
  p.cosp = cosp; p.sinp = sinp; p.positions = positions;
  p.c = cache_params(cache, page_table, lengths);
  p.o = o;
  p.sums = ws;
  p.stats = ws + w.stats;
  p.owners = reinterpret_cast<int*>(ws + w.owners);
  p.B = desc->seqs; p.H = desc->heads; p.Hkv = desc->kv_heads; p.n_pos = desc->n_pos; p.has_cls = desc->has_cls;
  p.workers = workers;
  p.direct = w.total == 0;
  p.window = window; p.sinks = sinks;
  p.g_tiles = decode_tiles(desc);
  p.c2 = desc->softmax_scale * 1.4426950408889634f;
  return launch_rc(launch_decode(p, desc->dtype, desc->head_dim, static_cast<hipStream_t>(stream)));
}

// Several new tokens per sequence over a cache (tree.hip).  The host knows the sequences' number, their
// mean of new tokens and their room alone.
int tree_group(const farope_seq_desc* d) { return d->heads / d->kv_heads; }
// Rows of a tile: 128 read the cache half as often, once a sequence's rows do not fit 64.  Measured, us with 64 and
// with 128 (32 sequences of 8192 rows, 32 heads of 8, D 128, bf16): 16 new tokens each (64 rows) 243, 249; 20 279, 250;
// 32 283, 256; 48 638, 345.
int tree_rows(const farope_seq_desc* d) {
  return d->dtype != FAROPE_F32 && (int64_t)d->tokens * tree_group(d) / d->seqs > 64 ? 128 : 64;
}
int64_t tree_slots(const farope_seq_desc* d) { return (int64_t)d->tokens * tree_group(d) / tree_rows(d) + d->seqs + 1; }
int tree_stage(const farope_seq_desc* d) { return d->head_dim * elem_size(d->dtype) <= 128 ? 64 : 32; }   // (kTreeRows of tree.hip)
// A workgroup a tile instead of even shares and a join: where sequences are short their lengths differ by little, and
// the join's launch is what costs.  Measured, us with shares and alone (8 new tokens, 12 heads, D 64, bf16): one sequence of
// 120 rows 12.4, 9.2, of 500 13.4, 12.9, of 1000 14.4, 18.9; 64 of 500 43, 32.  32 new tokens, 32 heads of 8, D 128: 32 of 480
// 43, 34, but 64 of 250 41, 51 (a second round of workgroups, mostly their starts); 32 of unlike lengths up to 8192 150, 254.
bool tree_direct(const farope_seq_desc* d, const farope_cache_desc* c) {
  return (int64_t)c->max_pages * c->page_rows <= 512;
}
// Workgroups of a key head: two a CU, one for rows of more than 256 bytes; that is one resident round from D 64 on.  Measured, us with half
// of it, all, two (32 heads of 8, D 128, bf16): 8 sequences of 4096 rows, 16 new tokens 50, 48, 61; 32 of 8192, 32 new 264, 259, 289.
// At D 32 a CU holds three and four; with two, three, four: 32 of 4096, 16 new 53.8, 55.0, 59.2, 8 of 4096 26.5, 29.0, 26.7, 4 of 8192,
// 512 new, fp16 142.8, 142.7, 139.6.
int tree_workers(const farope_seq_desc* d, const farope_cache_desc* c) {
  const int64_t room = ((int64_t)c->max_pages * c->page_rows + tree_stage(d) - 1) / tree_stage(d);
  const int64_t wgs = (int64_t)kCus * (d->head_dim * elem_size(d->dtype) <= 256 ? 2 : 1);
  int64_t n = wgs / d->kv_heads;
  if (n < 1) n = 1;
  const int64_t most = tree_slots(d) * ((room + kTreeLeast - 1) / kTreeLeast);
  return (int)(n < most ? n : most);
}
// Workspace, in fp32 elements, each part from a 16-byte boundary: sums, their statistics, owners.
struct TreeWs {
  int64_t stats, owners, total;
};
TreeWs tree_ws(const farope_seq_desc* d, const farope_cache_desc* c) {
  if (tree_direct(d, c)) return TreeWs{};
  const int64_t rows = 2 * (int64_t)tree_workers(d, c) * d->kv_heads * tree_rows(d);
  TreeWs w{};
  w.stats = rows * d->head_dim;
  w.owners = w.stats + 2 * rows;
  w.total = w.owners + 4 * tree_slots(d);
  return w;
}

// The cache of a call that moves rows as they are: no queries, no tables.
int check_rows(const farope_seq_desc* d) {
  if (!d) return FAROPE_ERR_NULL;
  if (d->seqs < 1 || d->kv_heads < 1) return FAROPE_ERR_SHAPE;
  if (d->head_dim != 32 && d->head_dim != 64 && d->head_dim != 128 && d->head_dim != 256) return FAROPE_ERR_HEAD_DIM;
  if (d->dtype != FAROPE_F32 && d->dtype != FAROPE_F16 && d->dtype != FAROPE_BF16) return FAROPE_ERR_DTYPE;
  return (int64_t)d->kv_heads * d->head_dim > (int64_t(1) << 24) ? FAROPE_ERR_SHAPE : FAROPE_OK;
}
int row_chunks(const farope_seq_desc* d) { return d->head_dim * elem_size(d->dtype) / 16; }
constexpr int kMaxPath = 2048;   // columns of a path (cache_accept_kernel: 8 rows a thread)

// Workspace, in fp32 elements, each part from a 16-byte boundary.
struct ForkWs {
  int64_t free, table, wanted, len, from, list, total;
};
int fork_chunks(const farope_cache_desc* c) { return (c->pages + kForkChunk - 1) / kForkChunk; }
ForkWs fork_ws(int32_t seqs, const farope_cache_desc* c) {
  auto al = [](int64_t x) { return (x + 3) & ~int64_t(3); };
  const int64_t chunks = fork_chunks(c), entries = (int64_t)seqs * c->max_pages;
  ForkWs w{};
  w.free = chunks * (kForkChunk / 32);
  w.table = w.free + al(chunks);
  w.wanted = w.table + al(entries);
  w.len = w.wanted + al(seqs);
  w.from = w.len + al(seqs);
  w.list = w.from + al(seqs);
  w.total = w.list + al(entries < c->pages ? entries : c->pages);
  return w;
}

}  // namespace

extern "C" {

int farope_seq_streams(const farope_seq_desc* desc, const void* x, const int64_t stride[3]) {
  return check_desc(desc, false) == FAROPE_OK && stride && streams(desc, x, stride);
}

size_t farope_seq_workspace_elems(const farope_seq_desc* desc, int32_t backward, int32_t v_streams, int32_t dout_streams) {
  if (check_desc(desc, true) != FAROPE_OK) return 0;
  return (size_t)seq_ws(desc, backward != 0, v_streams != 0, dout_streams != 0, Window{0, 0}).total;
}

size_t farope_seq_window_workspace_elems(const farope_seq_desc* desc, int32_t window, int32_t sinks, int32_t backward,
                                         int32_t v_streams, int32_t dout_streams) {
  if (check_desc(desc, true) != FAROPE_OK || window < 1 || sinks < 0) return 0;
  return (size_t)seq_ws(desc, backward != 0, v_streams != 0, dout_streams != 0, window_of(desc, window, sinks)).total;
}

int farope_seq_fwd(const farope_seq_desc* desc, const void* q, const int64_t q_stride[3], const void* k,
                   const int64_t k_stride[3], const void* v, const int64_t v_stride[3], const float* cosp, const float* sinp,
                   const int32_t* positions, const int32_t* cu, void* o, float* lse, float* ws, size_t ws_elems, void* stream) {
  return seq_fwd_call(desc, Window{0, 0}, q, q_stride, k, k_stride, v, v_stride, cosp, sinp, positions, cu, o, lse, ws, ws_elems, stream);
}

int farope_seq_bwd(const farope_seq_desc* desc, const void* q, const int64_t q_stride[3], const void* k,
                   const int64_t k_stride[3], const void* v, const int64_t v_stride[3], const void* o, const void* dout,
                   const int64_t dout_stride[3], const float* lse, const float* cosp, const float* sinp,
                   const int32_t* positions, const int32_t* cu, void* dq, void* dk, void* dv, float* ws, size_t ws_elems,
                   void* stream) {
  return seq_bwd_call(desc, Window{0, 0}, q, q_stride, k, k_stride, v, v_stride, o, dout, dout_stride, lse, cosp, sinp, positions, cu, dq, dk, dv, ws, ws_elems, stream);
}

int farope_seq_window_fwd(const farope_seq_desc* desc, int32_t window, int32_t sinks, const void* q, const int64_t q_stride[3], const void* k,
                          const int64_t k_stride[3], const void* v, const int64_t v_stride[3], const float* cosp, const float* sinp,
                          const int32_t* positions, const int32_t* cu, void* o, float* lse, float* ws, size_t ws_elems, void* stream) {
  FAROPE_TRY(check_desc(desc, true));
  if (window < 1 || sinks < 0) return FAROPE_ERR_SHAPE;
  const farope_seq_desc causal = causal_desc(desc);
  return seq_fwd_call(&causal, window_of(desc, window, sinks), q, q_stride, k, k_stride, v, v_stride, cosp, sinp, positions, cu, o, lse, ws, ws_elems, stream);
}

int farope_seq_window_bwd(const farope_seq_desc* desc, int32_t window, int32_t sinks, const void* q, const int64_t q_stride[3], const void* k,
                          const int64_t k_stride[3], const void* v, const int64_t v_stride[3], const void* o, const void* dout,
                          const int64_t dout_stride[3], const float* lse, const float* cosp, const float* sinp,
                          const int32_t* positions, const int32_t* cu, void* dq, void* dk, void* dv, float* ws, size_t ws_elems,
                          void* stream) {
  FAROPE_TRY(check_desc(desc, true));
  if (window < 1 || sinks < 0) return FAROPE_ERR_SHAPE;
  const farope_seq_desc causal = causal_desc(desc);
  return seq_bwd_call(&causal, window_of(desc, window, sinks), q, q_stride, k, k_stride, v, v_stride, o, dout, dout_stride, lse, cosp, sinp, positions, cu, dq, dk, dv, ws, ws_elems, stream);
}

int farope_cache_append(const farope_seq_desc* desc, const void* k, const int64_t k_stride[3], const void* v,
                        const int64_t v_stride[3], const float* cosp, const float* sinp, const int32_t* positions,
                        const farope_cache_desc* cache, const int32_t* page_table, const int32_t* lengths, const int32_t* cu,
                        void* stream) {
  FAROPE_TRY(check_desc(desc, false));
  if (!cu && desc->tokens != desc->seqs) return FAROPE_ERR_SHAPE;
  if (desc->tokens == 0) return FAROPE_OK;
  if (!k_stride || !v_stride) return FAROPE_ERR_NULL;
  const int es = elem_size(desc->dtype);
  FAROPE_TRY(check_ptr(k, es));
  FAROPE_TRY(check_ptr(v, es));
  FAROPE_TRY(check_ptr(cosp, 16));
  FAROPE_TRY(check_ptr(sinp, 16));
  if (positions) FAROPE_TRY(check_ptr(positions, 4));
  if (cu) FAROPE_TRY(check_ptr(cu, 4));
  FAROPE_TRY(check_cache(desc, cache, page_table, lengths));
  if (token_blocks(desc) > kMaxWorkgroups) return FAROPE_ERR_SHAPE;
  AppendParams p{};
  p.k = k; p.v = v;
  for (int i = 0; i < 3; ++i) { p.sk[i] = k_stride[i]; p.sv[i] = v_stride[i]; }
  p.vec_k = vec_rows(k, k_stride, es); p.vec_v = vec_rows(v, v_stride, es);
  p.cosp = cosp; p.sinp = sinp; p.positions = positions; p.cu = cu;
  p.c = cache_params(cache, page_table, lengths);
  p.T = desc->tokens; p.B = desc->seqs; p.Hkv = desc->kv_heads; p.n_pos = desc->n_pos; p.has_cls = desc->has_cls;
  return launch_rc(launch_cache_append(p, desc->dtype, desc->head_dim, static_cast<hipStream_t>(stream)));
}

size_t farope_decode_workspace_elems(const farope_seq_desc* desc, const farope_cache_desc* cache) {
  if (check_desc(desc, true) != FAROPE_OK || !cache || cache->max_pages < 1 || cache->page_rows < 1) return 0;
  return (size_t)decode_ws(desc, cache, 0, 0).total;
}

size_t farope_decode_window_workspace_elems(const farope_seq_desc* desc, const farope_cache_desc* cache, int32_t window,
                                            int32_t sinks) {
  if (check_desc(desc, true) != FAROPE_OK || !cache || cache->max_pages < 1 || cache->page_rows < 1 || window < 1 || sinks < 0)
    return 0;
  return (size_t)decode_ws(desc, cache, decode_window(cache, window), sinks).total;
}

int farope_decode(const farope_seq_desc* desc, const void* q, const int64_t q_stride[3], const float* cosp, const float* sinp,
                  const int32_t* positions, const farope_cache_desc* cache, const int32_t* page_table, const int32_t* lengths,
                  void* o, float* ws, size_t ws_elems, void* stream) {
  return decode_call(desc, 0, 0, q, q_stride, cosp, sinp, positions, cache, page_table, lengths, o, ws, ws_elems, stream);
}

int farope_decode_window(const farope_seq_desc* desc, int32_t window, int32_t sinks, const void* q, const int64_t q_stride[3],
                         const float* cosp, const float* sinp, const int32_t* positions, const farope_cache_desc* cache,
                         const int32_t* page_table, const int32_t* lengths, void* o, float* ws, size_t ws_elems, void* stream) {
  if (window < 1 || sinks < 0) return FAROPE_ERR_SHAPE;
  if (!cache) return FAROPE_ERR_NULL;
  return decode_call(desc, decode_window(cache, window), sinks, q, q_stride, cosp, sinp, positions, cache, page_table, lengths, o, ws,
                     ws_elems, stream);
}
size_t farope_tree_workspace_elems(const farope_seq_desc* desc, const farope_cache_desc* cache) {
  if (check_desc(desc, true) != FAROPE_OK || !cache || cache->max_pages < 1 || cache->page_rows < 1) return 0;
  return (size_t)tree_ws(desc, cache).total;
}

int farope_tree(const farope_seq_desc* desc, const void* q, const int64_t q_stride[3], const float* cosp, const float* sinp,
                const int32_t* positions, const farope_cache_desc* cache, const int32_t* page_table, const int32_t* lengths,
                const int32_t* cu, const uint8_t* tree, int64_t tree_stride, int32_t tree_cols, void* o, float* ws, size_t ws_elems,
                void* stream) {
  FAROPE_TRY(check_desc(desc, true));
  if (desc->tokens == 0) return FAROPE_OK;
  if (!q_stride) return FAROPE_ERR_NULL;
  const int es = elem_size(desc->dtype);
  FAROPE_TRY(check_ptr(q, es));
  FAROPE_TRY(check_ptr(cosp, 16));
  FAROPE_TRY(check_ptr(sinp, 16));
  if (positions) FAROPE_TRY(check_ptr(positions, 4));
  FAROPE_TRY(check_cache(desc, cache, page_table, lengths));
  FAROPE_TRY(check_ptr(cu, 4));
  // (the rows of a sequence's tree are reached by 32-bit offsets)
  if (tree && (tree_cols < 0 || tree_stride < 0 || tree_stride > INT32_MAX || tree_stride * desc->tokens + tree_cols > INT32_MAX))
    return FAROPE_ERR_SHAPE;
  FAROPE_TRY(check_ptr(o, 16));
  const TreeWs w = tree_ws(desc, cache);
  if (w.total) {
    FAROPE_TRY(check_ptr(ws, 16));
    if ((int64_t)ws_elems < w.total) return FAROPE_ERR_SCRATCH;
  }
  TreeParams p{};
  p.q = q;
  for (int i = 0; i < 3; ++i) p.sq[i] = q_stride[i];
  p.vec_q = vec_rows(q, q_stride, es);
  p.cosp = cosp; p.sinp = sinp; p.positions = positions; p.cu = cu;
  p.tree = tree; p.stree = tree_stride; p.cols = tree_cols;
  p.c = cache_params(cache, page_table, lengths);
  p.o = o;
  p.sums = ws;
  p.stats = ws + w.stats;
  p.owners = reinterpret_cast<int*>(ws + w.owners);
  p.T = desc->tokens; p.B = desc->seqs; p.H = desc->heads; p.Hkv = desc->kv_heads; p.n_pos = desc->n_pos; p.has_cls = desc->has_cls;
  for (int i = 0; i < 2; ++i) {
    const int64_t k = cache->k_stride[i] * es / 16, v = cache->v_stride[i] * es / 16;
    if (k < 0 || v < 0 || k > UINT32_MAX || v > UINT32_MAX) return FAROPE_ERR_SHAPE;
    p.k16[i] = (uint32_t)k;
    p.v16[i] = (uint32_t)v;
  }
  p.alike = p.k16[0] == p.v16[0] && p.k16[1] == p.v16[1];
  // With 2^(l-1) < page <= 2^l, m = floor(2^(31+l) / page) + 1 and e = m page - 2^(31+l) in (0, page]: x m / 2^(31+l) =
  // x / page + x e / (page 2^(31+l)), and x e < 2^31 2^l, so the second part is less than 1 / page.
  int l = 0;
  while (l < 31 && (int64_t(1) << l) < cache->page_rows) ++l;
  p.page_mul = (uint32_t)(((uint64_t(1) << (31 + l)) / (uint64_t)cache->page_rows + 1));
  p.page_shift = 31 + l;
  p.rows = tree_rows(desc);
  // (rows of a key head in 32 bits, with a tile's more; workgroups: a tile each, and in the join 16 rows each)
  const int64_t join = w.total ? p.rows / 16 : 1;
  if ((int64_t)p.T * p.H > INT32_MAX - 256 || tree_slots(desc) * p.Hkv * join > kMaxWorkgroups) return FAROPE_ERR_SHAPE;
  p.slots = (int)tree_slots(desc);
  p.workers = tree_workers(desc, cache);
  p.direct = w.total == 0;
  p.c2 = desc->softmax_scale * 1.4426950408889634f;
  if (!p.direct && (int64_t)p.workers * p.Hkv > kMaxWorkgroups) return FAROPE_ERR_SHAPE;
  return launch_rc(launch_tree(p, desc->dtype, desc->head_dim, static_cast<hipStream_t>(stream)));
}

int farope_cache_accept(const farope_seq_desc* desc, const farope_cache_desc* cache, const int32_t* page_table,
                        const int32_t* lengths, const int32_t* path, int64_t path_stride, int32_t path_cols, int32_t* new_lengths,
                        void* stream) {
  FAROPE_TRY(check_rows(desc));
  FAROPE_TRY(check_cache(desc, cache, page_table, lengths));
  if (path_cols < 0 || path_cols > kMaxPath || path_stride < 0) return FAROPE_ERR_SHAPE;
  if (path_cols) FAROPE_TRY(check_ptr(path, 4));
  FAROPE_TRY(check_ptr(new_lengths, 4));
  AcceptParams p{};
  p.c = cache_params(cache, page_table, lengths);
  p.path = path; p.spath = path_stride; p.cols = path_cols;
  p.out = new_lengths;
  p.B = desc->seqs; p.Hkv = desc->kv_heads; p.es = elem_size(desc->dtype); p.cpr = row_chunks(desc);
  if ((int64_t)p.B * 2 * p.Hkv * p.cpr > kMaxWorkgroups) return FAROPE_ERR_SHAPE;   // (one chunk a workgroup at least)
  return launch_rc(launch_cache_accept(p, static_cast<hipStream_t>(stream)));
}

size_t farope_cache_fork_workspace_elems(int32_t seqs, const farope_cache_desc* cache) {
  if (seqs < 1 || !cache || cache->pages < 1 || cache->max_pages < 1) return 0;
  return (size_t)fork_ws(seqs, cache).total;
}

int farope_cache_fork(const farope_seq_desc* desc, const farope_cache_desc* cache, int32_t* page_table, int32_t* lengths,
                      int32_t* refs, const int32_t* parents, const int32_t* room, int32_t* missing, float* ws, size_t ws_elems,
                      void* stream) {
  FAROPE_TRY(check_rows(desc));
  FAROPE_TRY(check_cache(desc, cache, page_table, lengths));
  if (desc->seqs > 1 && cache->table_stride < cache->max_pages) return FAROPE_ERR_SHAPE;   // (rows are written)
  FAROPE_TRY(check_ptr(refs, 4));
  FAROPE_TRY(check_ptr(parents, 4));
  if (room) FAROPE_TRY(check_ptr(room, 4));
  FAROPE_TRY(check_ptr(missing, 4));
  FAROPE_TRY(check_ptr(ws, 16));
  const ForkWs w = fork_ws(desc->seqs, cache);
  if ((int64_t)ws_elems < w.total) return FAROPE_ERR_SCRATCH;
  ForkParams p{};
  p.c = cache_params(cache, page_table, lengths);
  p.pages = page_table; p.lengths = lengths; p.refs = refs; p.parents = parents; p.room = room; p.missing = missing;
  int32_t* const ints = reinterpret_cast<int32_t*>(ws);
  p.bits = reinterpret_cast<uint64_t*>(ws);
  p.free = ints + w.free; p.table = ints + w.table; p.wanted = ints + w.wanted; p.len = ints + w.len; p.from = ints + w.from;
  p.list = ints + w.list;
  p.chunks = fork_chunks(cache);
  p.B = desc->seqs; p.Hkv = desc->kv_heads; p.es = elem_size(desc->dtype); p.cpr = row_chunks(desc);
  const int64_t row = (int64_t)p.Hkv * p.cpr, chunks = 2 * (int64_t)p.c.page * row;
  if ((int64_t)p.B * p.c.max_pages > INT32_MAX || (int64_t)p.c.page * row > INT32_MAX ||
      (chunks / 2048 + 2) * p.B > kMaxWorkgroups || (int64_t)p.B + p.chunks > kMaxWorkgroups)
    return FAROPE_ERR_SHAPE;
  return launch_rc(launch_cache_fork(p, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
