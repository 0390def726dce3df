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
  static constexpr int kSmem = (4 + kRing) * kTile;
  static_assert(128 * HD * 4 <= 2 * kTile, "the results of 128 rows pass through the memory of their q");
  static_assert(kSmem + 2048 <= 227 * 1024, "shared memory");
};
inline int tc_block(int kind) { return kind == kKvBf16 ? 128 : 64; }
constexpr int kTcExps = 128;  // bytes of a K or V block's powers per slot
// Scratch of a (KV head, block) pair: K and V as fp16 planes; behind those of all pairs the powers per slot,
// then 4 bytes each of what the main kernel is told of them.
constexpr size_t tc_unit_bytes(int hd) { return (size_t)2 * 128 * 2 * hd + 2 * kTcExps + 4; }

cudaError_t configure_rows_attn_tc();
// Long chunks of a batch; a.planes has room for their (KV head, block) pairs.
cudaError_t launch_rows_tc(const RowsAttnArgs& a, const RowsBatch& b, int kind, int hd, int sms, int* launches,
                           cudaStream_t st);

}  // namespace dllm
