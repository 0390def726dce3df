// rows_attn_tc.cuh — the tile shapes of rows_attn_tc.cu, for the host that cuts a batch into
// tiles, and its launchers.
#pragma once

#include "rows_attn.cuh"

namespace dllm {

constexpr int kTcSoftWarps = 8, kTcSoft = 32 * kTcSoftWarps;  // the softmax's share
constexpr int kTcThreads = kTcSoft + 128;
constexpr int kTcTileRows = 256;  // rows of a CTA
constexpr int kTcRing = 6, kTcTurns = 3;  // tiles of the ring at most, and half as many

template <int KIND, int HD>
struct TcTile {
  static constexpr int kPlanes = KIND == kKvBf16 ? 1 : 2;
  static constexpr int BN = 128 / kPlanes;               // slots of a block
  static constexpr int BOX = HD / 64;                    // 64-dim boxes
  static constexpr int kBox = 128 * 128;                 // bytes of 128 rows of a box
  static constexpr int kTile = BOX * kBox;               // of a K or V block, and of one term of 128 rows of q
  static constexpr int kRing = HD == 64 ? 6 : 3;         // K and V blocks under way
  static constexpr int kTurns = (kRing + 1) / 2;
  static constexpr int kOut = kTcTileRows * (HD + 6) * 4;  // the results, over q and the ring
  static constexpr int kSmem = (4 + kRing) * kTile;
  static_assert(kOut <= (4 + kRing) * kTile, "results reuse the operands' memory");
  static_assert(kSmem + 2048 <= 227 * 1024, "shared memory");
};
inline int tc_block(int kind) { return kind == kKvBf16 ? 128 : 64; }

// All tiles of 256 rows of a batch (sequence by sequence, KV head by KV head), and their blocks
// one after the other, cut into equal shares: CTA c takes `share` blocks from block
// begin_block[c] of tile begin_tile[c] on. A tile in one CTA's share is written out; of the
// others each CTA leaves partial results, at most two of 256 rows (its first segment's, and its
// last one's), which are joined.
constexpr int kTcMaxCtas = 192;
struct RowsTcArgs {
  RowsAttnArgs a;
  int n_seqs, share, total;
  int seq[kRowsMaxSeqs], row0[kRowsMaxSeqs], m[kRowsMaxSeqs], t0[kRowsMaxSeqs];
  int tile0[kRowsMaxSeqs + 1];  // tiles before the sequence
  int unit0[kRowsMaxSeqs + 1];  // (KV head, block) pairs before the sequence
  int begin_tile[kTcMaxCtas], begin_block[kTcMaxCtas];
  int split_tile[kTcMaxCtas], split_cta[kTcMaxCtas], split_n[kTcMaxCtas];  // joined tiles, their first CTA, CTAs
};
static_assert(sizeof(RowsTcArgs) <= 8192, "kernel arguments");

// One tile, its sequence and KV head.
struct RowsTcTile {
  int i, seq, row0, m, t0, head, G, r0, R;
  RowsView v;
  __host__ __device__ static int tiles_of(int m, int G) { return (m * G + kTcTileRows - 1) / kTcTileRows; }
  DLLM_DEV RowsTcTile(const RowsTcArgs& P, int tile, int bn) : v(0, 0, 1, 0, 1) {
    i = rows_find(P.tile0, P.n_seqs, tile);
    seq = P.seq[i], row0 = P.row0[i], m = P.m[i], t0 = P.t0[i];
    G = P.a.nq / P.a.pages.kvh, R = m * G;
    const int tiles = tiles_of(m, G), at = tile - P.tile0[i];
    head = at / tiles;
    r0 = at % tiles * kTcTileRows;
    const int last = (r0 + kTcTileRows < R ? r0 + kTcTileRows : R) - 1;
    v = RowsView(t0 + r0 / G, t0 + last / G, P.a.window, P.a.sinks, bn);
  }
  DLLM_DEV int slot_of(int r) const { return r < R ? t0 + r / G : -1; }
  DLLM_DEV int place(int r, int nq) const { return r / G * nq + head * G + r % G; }
};

cudaError_t configure_rows_attn_tc();
// Long chunks of a batch; a.planes holds their (KV head, block) pairs, 2 x 256 x head-size bytes
// each, and 16 bytes each behind.
cudaError_t launch_rows_tc(const RowsAttnArgs& a, const RowsBatch& b, int kind, int hd, int sms, int* launches,
                           cudaStream_t st);

}  // namespace dllm
