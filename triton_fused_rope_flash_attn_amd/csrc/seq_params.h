// Kernel argument blocks and launchers of attention over packed sequences and
// over a paged cache (seq_api.hip calls them).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace farope {

constexpr int kSeqNW = 4;                  // waves per workgroup
constexpr int kSeqThreads = 64 * kSeqNW;

// Token t, head h, channel d of an input: t*s[0] + h*s[1] + d*s[2] elements.
struct SeqParams {
  const void* q;
  const void* k;
  const void* v;
  const void* dout;
  int64_t sq[3], sk[3], sv[3], sdo[3];
  int vec_q, vec_k, vec_v, vec_do;   // 16-byte access (seq_api.hip: vec_rows)
  const float* cosp;                 // [n_pos, D/2]
  const float* sinp;
  const int* positions;              // [T] table rows, or null: by index
  const int* cu;                     // [B + 1]
  void* o;                           // [T, H, D]
  float* lse;                        // [H, T], natural log
  void* dq;                          // [T, H, D]
  void* dk;                          // [T, Hkv, D]
  void* dv;
  // workspace
  void* khat;                        // [Hkv, T, D]: rotated K rows times scale * log2 e; null: no such pass
  void* vcopy;                       // [Hkv, T, D]: V, where its own rows cannot be streamed (else null)
  void* qhat;                        // [H, T, D]: rotated Q rows
  void* gcopy;                       // [H, T, D]: dO, where its own rows cannot be streamed (else null)
  int* map_q;                        // [slots][4]: the tiles of the query kernels' workgroups (SeqTile); null: none
  int* map_k;                        // and of the key kernel's
  float* nl;                         // [H, T]: -LSE * log2 e (fp16: and kWeightUp)
  float* nd;                         // [H, T]: -rowsum(dO * O)
  float* ng;                         // [H, T]: norms of dO's rows (fp16 at head_dim 128)
  float* pk;                         // [parts, T, Hkv, D]: sums of the parts of dK / scale (rotated), parts > 1
  float* pv;                         // and of dV
  int parts;                         // parts of a key tile's queries
  int T, B, H, Hkv, n_pos, has_cls, causal;
  float scale, c2;                   // softmax scale; times log2 e
  int slots;                         // row slots of the launch (set by the launcher)
};

// A slot per 2^lb rows, one more per sequence, and the tokens behind the last one.
inline int64_t seq_slots(int T, int B, int lb) { return (int64_t)(T >> lb) + B + 1; }

// Rows per workgroup of the forward and of dQ, 128 (two 16-row subtiles per wave) or 64.  Two
// subtiles halve the LDS reads per product, but cost workgroups, and products above the
// diagonal.  ("24 up to 2048": here and beside the kernels lengths drawn down to a 16th of the longest, on a
// logarithmic scale; these have a mean of 943.)  16-bit tensors; measured (us, forward and backward, 64 / 128 rows; "sequences x
// tokens, heads" and the call's 128-row tiles), D 128: 24 up to 2048, 16 [2828] 916 / 869, 1 x 16384, 8
// [1024] 2702 / 2512, 4 up to 4096, 8 [676] 455 / 484, 1 x 4096, 16 [512] 422 / 467, 8 x 1024, 8 [512]
// 164 / 175, 64 up to 200, 8 [308] 89 / 105.  Forward, D 64: 1 x 8192, 16 [1024] 170 / 152, 1 x 4096, 16
// [512] 57 / 70, 16 up to 2048, 16 [2248] 99 / 104, 8 x 1024, 16 [1024] 43 / 49; D 32: 4 x 8192, 8 [2048]
// 235 / 214, 4 x 2048, 8 [512] 34.8 / 36.3.  D 256, forward and backward: 2 x 4096, 8 [512] 1242 / 1173, 16 x
// 512, 8 [512] 333 / 331, 4 x 1024, 8 [256] 268 / 302, 64 up to 200 (77), 12 [462] 296 / 368, 125 up to 149 (54),
// 8 [423] 292 / 365.
inline int seq_tile_rows(int T, int B, int H, int D, bool f32) {
  const int64_t tiles = (int64_t)T * H / 128, mean = T / B;
  if (f32) return 64;
  if (D == 256) return tiles >= 2 * 256 && mean >= 256 ? 128 : 64;
  if (D == 128) return tiles >= 4 * 256 && mean >= 256 ? 128 : 64;
  return tiles >= 4 * 256 && mean >= 4096 ? 128 : 64;
}

// Whether the workgroups of a causal call come in the order of their work, over all sequences, not
// sequence by sequence (whose tiles then read K and V from L2 one after the other: better for short
// ones).  Measured (us, by sequence / by work; "sequences up to tokens (mean), heads"), forward, D
// 128: 24 up to 2048 (943), 16 210 / 190, 8 up to 8192, 8 452 / 413, 32 up to 512 (228), 16 51 / 46; D 64: 16
// up to 2048 (1124), 16 103 / 98, 8 x 1024, 16 43.8 / 41.7, 64 up to 577 (223), 12 40 / 49.  Forward
// and backward: 1020 / 894, 2496 / 2115, 203 / 187, 426 / 421, 149 / 154; 200 up to 600 (224), 8 324 / 344.
constexpr int kOrderSeqs = 256;   // (four sequences per lane of the search)
inline int seq_order(int T, int B, int D, int causal) {
  return causal && B > 1 && B <= kOrderSeqs && T / B >= (D >= 128 ? 128 : 512);
}

hipError_t launch_seq_prep(const SeqParams& p, int dt, int D, bool backward, hipStream_t st);
hipError_t launch_seq_fwd(const SeqParams& p, int dt, int D, hipStream_t st);
hipError_t launch_seq_bwd(const SeqParams& p, int dt, int D, hipStream_t st);

// Paged cache: row r of page g, key head h: g*s[0] + r*s[1] + h*s[2] elements,
// channels contiguous, every row 16-byte aligned.
struct CacheParams {
  void* kc;
  void* vc;
  int64_t skc[3], svc[3];
  const int* pages;      // [B, max_pages]
  int64_t spages;        // elements between its rows
  const int* lengths;    // [B]
  int n_pages, page, max_pages;
};

struct AppendParams {
  const void* k;
  const void* v;
  int64_t sk[3], sv[3];
  int vec_k, vec_v;
  const float* cosp;
  const float* sinp;
  const int* positions;  // [T], or null
  const int* cu;         // [B + 1], or null: token t is sequence t's
  CacheParams c;
  int T, B, Hkv, n_pos, has_cls;
};
hipError_t launch_cache_append(const AppendParams& p, int dt, int D, hipStream_t st);

struct DecodeParams {
  const void* q;
  int64_t sq[3];         // sequence, head, channel
  int vec_q;
  const float* cosp;
  const float* sinp;
  const int* positions;  // [B], or null
  CacheParams c;
  void* o;               // [B, H, D]
  float* sums;           // [workers + B, H, D]: unnormalised O of (worker, sequence) pairs
  float* stats;          // [workers + B, H, 2]: their max logit (log2 units) and row sum
  int* owners;           // [B, 2]: a sequence's first worker, and how many have a part of it
  int B, H, Hkv, n_pos, has_cls;
  int workers;           // workgroups of a key head and query tile
  int direct;            // worker i has sequence i: nothing is joined
  int g_tiles;           // tiles of 16 query heads in a group
  float c2;
};
// Workers of a call: decode_workers in seq_api.hip.
hipError_t launch_decode(const DecodeParams& p, int dt, int D, hipStream_t st);

}  // namespace farope
