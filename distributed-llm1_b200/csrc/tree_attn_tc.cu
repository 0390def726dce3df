// tree_attn_tc.cu — tree attention over a bf16 cache on the tcgen05 tensor cores, for
// trees whose rows (nodes x query heads of a KV head) are worth a 128-row tile.
//
// The mathematics and the precision are tree_attn.cu's: q and p are cut into three
// bf16 terms, and each product runs smallest terms first into one fp32 accumulator, so
// that only the last pass adds at full size (the tensor core truncates each addition);
// a block's p . V starts from zero and is added to the running output in registers.
//
// One CTA, three warpgroups, one 128-row tile over its share of the 64-slot blocks, which
// it takes in pairs:
//   producer (1 warp)    TMA: K of a pair, V of a block (128-byte swizzle) into rings
//   MMA (1 warp)         S = q K^T of a pair (128 slots at once), O = P V of a block by halves
//                        of 64 dims
//   helper (1 warp)      the blocks that hold drafted rows: rows behind the last node are
//                        zeroed and non-finite values taken out before the MMA reads V
//   two softmax groups   128 threads, one row each; group w takes the pair's block w with a
//                        maximum, sum and output of its own: S from tensor memory, online
//                        softmax, P back as three bf16 planes (the MMA's A operand is read
//                        from tensor memory), then O into its registers
// The groups' results are joined like two splits. Tensor memory (512 columns): S of two pairs
// 2 x 128, P 2 x 96, O 64. The MMA warp runs the scores two pairs ahead, a quarter of a pair
// after each half of O, so that O is read while the scores keep the tensor core busy and
// the softmax of a block has a whole pair's time. V is read as it lies, slots x dims: a
// descriptor with the dims as the contiguous ("MN") direction.
// Bound: per pair 24 MMAs of 128 x 128 x 16 from shared memory (65 cycles) and 48 of 128 x 64
// x 16 with A in tensor memory (33): 3150 cycles, 0.82 us per block of 64 slots, against 0.74
// us for its 64 x 512 bytes at one SM's share of HBM. Measured with clock stamps, 64 nodes x
// 7 heads at 32000 slots, 56 blocks per CTA, cold cache: 2370 cycles per block between the
// first S and the last O (1575 of MMAs), 10 500 cycles until the first S (1900 of them to set
// up barriers and tensor memory, the rest the first copies and the cut of q) and 10 000 from
// the last O to the end: 87, 7 and 6 % of the kernel. In the loop the scores' MMAs read 126
// of the 128 bytes that shared memory gives per cycle, so every barrier and every
// tensor-memory store of the softmax waits behind them, and a group's chain of softmax, P, O
// becomes the limit. (Scores block by block, 24 MMAs of N = 64, and O whole: a fifth more per
// block; a second issuing warp for O: 4 %.) With two blocks per CTA (13 nodes x 6 heads at 8191 slots)
// start, loop and end take 10 400, 9700 and 9300 cycles. The softmax threads spill 64 bytes
// at HD = 128.
#include "tree_attn_tc.cuh"

namespace dllm {
namespace {

constexpr int kTcAttnThreads = 384;
constexpr int kKStages = 2;    // pairs
constexpr int kVStages = 4;    // blocks
constexpr int kPair = 2 * kTcBlock;
template <int HD>
struct TcTile {
  static constexpr int BOX = HD / 64;                      // 64-dim boxes
  static constexpr int kQPlane = BOX * kTcRows * 128;      // bytes of one bf16 term of q
  static constexpr int kKBox = kPair * 128;                // bytes of 128 slots x 64 dims
  static constexpr int kVBox = kTcBlock * 128;             // bytes of 64 slots x 64 dims
  static constexpr int kK = BOX * kKBox, kV = BOX * kVBox; // bytes of a pair's K, a block's V
  static constexpr int kRing = kKStages * kK + kVStages * kV;
  static constexpr int kOut = 2 * kTcRows * (HD + 6) * 4;  // both groups' results, over q and rings
  static constexpr int kSmem = 1024 + 3 * kQPlane + kRing;
  static_assert(kOut <= 3 * kQPlane + kRing, "results reuse the operands' memory");
  static_assert(kSmem + 512 <= 227 * 1024, "shared memory");
  static constexpr int kQMma = 3 * BOX * 4;                // MMAs of a pair's scores
  static constexpr int kSteps = 2 * BOX;                   // halves of O per pair
  static constexpr uint32_t kP = 256, kO = 448;            // tensor-memory columns: S 0, 128; P; O
};

struct TcShared {
  uint64_t k_full[kKStages], k_empty[kKStages], v_full[kVStages], v_empty[kVStages];
  uint64_t s_full[2], s_free[2];               // per S buffer
  uint64_t p_ready[2], o_full[2], o_free[2];   // per softmax group
  uint64_t v_here[2], v_ok[2];                 // the (at most two) blocks with drafted rows
  uint64_t idle;                               // every MMA has completed
  uint32_t tmem;
  int bad[2];
  volatile int abort;
};

template <int HD>
__global__ void __launch_bounds__(kTcAttnThreads, 1)
    tree_attn_tc_kernel(const __grid_constant__ TAKernelArgs P, const __grid_constant__ CUtensorMap tmK,
                        const __grid_constant__ CUtensorMap tmV) {
  using T = TcTile<HD>;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) TcShared sh;
  const TreeAttnArgs& a = P.a;
  asm volatile("griddepcontrol.launch_dependents;");  // the join may be scheduled; it waits for this grid's end
  TATile k;
  k.sq = ta_seq(P, blockIdx.z);
  k.set_group(a.nq / a.kvh);
  k.head = blockIdx.y % a.kvh;
  k.r0 = (blockIdx.y / a.kvh) * kTcRows;
  k.R = k.sq.m * k.G;
  const int T0 = P.t0[blockIdx.z], slots = T0 + k.sq.m;
  k.nsplit = ta_splits(slots, kTcBlock, P.bps);
  k.split = blockIdx.x;
  if (k.r0 >= k.R || k.split >= k.nsplit) return;
  const int blk0 = k.split * P.bps;
  const int nb = min((slots + kTcBlock - 1) / kTcBlock, blk0 + P.bps) - blk0;
  const int np = (nb + 1) / 2;              // pairs
  const int draft0 = T0 / kTcBlock - blk0;  // the first block (of this CTA's) with drafted rows

  // the warp's number as a value that is the same in all its lanes by construction
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* sQ = base;
  unsigned char* sK = base + 3 * T::kQPlane;
  unsigned char* sV = sK + kKStages * T::kK;

  if (tid == 0) {
    for (int s = 0; s < kKStages; ++s) mbar_init(&sh.k_full[s], 1), mbar_init(&sh.k_empty[s], 1);
    for (int s = 0; s < kVStages; ++s) mbar_init(&sh.v_full[s], 1), mbar_init(&sh.v_empty[s], 1);
    for (int w = 0; w < 2; ++w) {
      mbar_init(&sh.s_full[w], 1), mbar_init(&sh.s_free[w], 256);
      mbar_init(&sh.p_ready[w], 128), mbar_init(&sh.o_full[w], 1), mbar_init(&sh.o_free[w], 128);
      mbar_init(&sh.v_here[w], 32), mbar_init(&sh.v_ok[w], 32);
      sh.bad[w] = 0;
    }
    mbar_init(&sh.idle, 1);
    sh.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // the pool rows of a block's boxes (lane 0 of the producer); boxes behind the end are
  // loaded again and not used
  const int page = 1 << a.kv.log2_page, box = page < kTcBlock ? page : kTcBlock;
  auto pool_row = [&](int n, int b) {
    const int slot = min((blk0 + n) * kTcBlock + b * box, slots - 1) & ~(box - 1);
    return a.tc_row0 + (a.kv.page_table[(size_t)k.sq.seq * a.kv.max_pages + (slot >> a.kv.log2_page)] * a.kvh + k.head) * page +
           (slot & (page - 1));
  };
  if (warp == 8) {
    if (lane == 0) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(&tmK) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&tmV) : "memory");
    }
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
  const unsigned long long anc = warp < 8 && k.r0 + (tid & 127) < k.R ? a.anc[k.sq.row0 + k.node_of(k.r0 + (tid & 127))] : 0ull;
  if (warp != 8) {
    // q, scaled so that the softmax is in powers of two, as three bf16 planes of swizzled
    // 64-dim boxes (what the K-major descriptor reads), while the producer's first copies fly.
    // Rows behind the last one stay as they are: a row of S, P and O comes from its row alone.
    constexpr int kWorkers = kTcAttnThreads - 32;
    ta_load_q<HD, kWorkers>(P, k, sQ, warp < 8 ? tid : tid - 32);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // q is read by the MMA
    asm volatile("bar.sync 2, %0;" ::"n"(kWorkers) : "memory");
  }

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 8 && lane == 0) {
      // ---- producer. The pools are one tensor of rows (layer, page, head, slot); a page holds 32
      // slots (two boxes of a block) or a multiple of 64 (one).
      int k_sent = 0, v_sent = 0;
      bool ok = true;  // nothing is loaded over memory that may still be read
      // K runs a pair ahead of V
      for (int j = 0; ok && j <= np; ++j) {
        if (j < np) {
          const int s = j % kKStages, blocks = min(2, nb - 2 * j);
          ok = wait_phase(&sh.k_empty[s], ((uint32_t)(j / kKStages) & 1u) ^ 1u, &sh.abort);
          if (!ok) break;
          mbar_expect_tx(&sh.k_full[s], blocks * T::kV);
          for (int h = 0; h < blocks; ++h)
            for (int b = 0; b < kTcBlock / box; ++b) {
              const int row = pool_row(2 * j + h, b);
              for (int x = 0; x < T::BOX; ++x)
                tma_load_2d(sK + s * T::kK + x * T::kKBox + (h * kTcBlock + b * box) * 128, &tmK, x * 64, row, &sh.k_full[s]);
            }
          k_sent = j + 1;
        }
        for (int n = max(0, 2 * (j - 1)); ok && n < min(nb, 2 * j); ++n) {
          const int s = n % kVStages;
          ok = wait_phase(&sh.v_empty[s], ((uint32_t)(n / kVStages) & 1u) ^ 1u, &sh.abort);
          if (!ok) break;
          mbar_expect_tx(&sh.v_full[s], T::kV);
          for (int b = 0; b < kTcBlock / box; ++b) {
            const int row = pool_row(n, b);
            for (int x = 0; x < T::BOX; ++x)
              tma_load_2d(sV + s * T::kV + x * T::kVBox + b * box * 128, &tmV, x * 64, row, &sh.v_full[s]);
          }
          v_sent = n + 1;
        }
      }
      // whatever happened to the others, the copies under way land before the CTA ends
      for (int j = max(0, k_sent - kKStages); j < k_sent; ++j)
        mbar_wait(&sh.k_full[j % kKStages], (uint32_t)(j / kKStages) & 1u);
      for (int j = max(0, v_sent - kVStages); j < v_sent; ++j)
        mbar_wait(&sh.v_full[j % kVStages], (uint32_t)(j / kVStages) & 1u);
    } else if (warp == 9) {
      // ---- MMA issuer. The whole warp runs the loop and one elected lane issues: the operands
      // of tcgen05.mma live in uniform registers, and in a branch on the lane number
      // every one of them was first moved there (130 to 230 cycles per MMA; 33 to 65 this way).
      const uint32_t leader = elect_one();
      const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kTcRows >> 4) << 24);  // fp32 += bf16 x bf16
      const uint32_t id_s = idesc | ((uint32_t)(kPair >> 3) << 17);            // N = 128 slots, K-major
      const uint32_t id_o = idesc | ((uint32_t)(64 >> 3) << 17) | (1u << 16);  // N = 64 dims, B with N contiguous
      // MMAs [from, to) of the scores of pair j, the lowest terms of q first
      auto scores = [&](int j, int from, int to) {
        const unsigned char* kb = sK + (j % kKStages) * T::kK;
#pragma unroll
        for (int i = 0; i < T::kQMma; ++i) {
          if (i < from || i >= to) continue;
          const int p = 2 - i / (T::BOX * 4), x = i / 4 % T::BOX, kk = i % 4;
          umma_bf16(tmem + (uint32_t)(j & 1) * kPair, umma_desc_sw128(sQ + p * T::kQPlane + x * (kTcRows * 128)) + 2ull * kk,
                    umma_desc_sw128(kb + x * T::kKBox) + 2ull * kk, id_s, (uint32_t)(i != 0));
        }
        if (to == T::kQMma) {
          umma_commit(&sh.k_empty[j % kKStages]);
          umma_commit(&sh.s_full[j & 1]);
        }
      };
      for (int j = 0; j < min(2, np); ++j) {
        wait_phase(&sh.k_full[j], 0u, &sh.abort);
        tc_fence_after();
        if (leader) scores(j, 0, T::kQMma);
        __syncwarp();
      }
      auto operands = [&](int n) {
        wait_phase(&sh.v_full[n % kVStages], (uint32_t)(n / kVStages) & 1u, &sh.abort);
        if (n >= draft0) {
          mbar_arrive(&sh.v_here[n - draft0]);
          wait_phase(&sh.v_ok[n - draft0], 0u, &sh.abort);
        }
        wait_phase(&sh.p_ready[n & 1], (uint32_t)(n >> 1) & 1u, &sh.abort);
      };
      operands(0);
      for (int j = 0; j < np; ++j) {
#pragma unroll
        for (int i = 0; i < T::kSteps; ++i) {
          const int w = i / T::BOX, h = i % T::BOX, n = 2 * j + w, s = n % kVStages;
          if (n < nb) {
            // O is free once its last half has been read
            const int last = i == 0 ? T::kSteps - 1 : i - 1, lj = i == 0 ? j - 1 : j;
            if (lj >= 0) wait_phase(&sh.o_free[last / T::BOX], (uint32_t)(lj * T::BOX + last % T::BOX) & 1u, &sh.abort);
            tc_fence_after();
            if (leader) {
#pragma unroll
              for (int p = 2; p >= 0; --p) {
                const uint32_t ap = tmem + T::kP + (uint32_t)w * 96 + (uint32_t)p * 32;
                const uint64_t bd = umma_desc_mn_sw128(sV + s * T::kV + h * T::kVBox, T::kVBox);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)  // 16 slots: 2048 bytes on
                  umma_bf16_ts(tmem + T::kO, ap + 8u * kk, bd + 128ull * kk, id_o, (uint32_t)(p != 2 || kk));
              }
              if (h == T::BOX - 1) umma_commit(&sh.v_empty[s]);
              umma_commit(&sh.o_full[w]);
            }
            __syncwarp();
          }
          // the next block's V and P, while the tensor core is busy
          if (h == T::BOX - 1 && n + 1 < nb) operands(n + 1);
          if (j + 2 < np) {
            if (i == 0) {
              wait_phase(&sh.k_full[j % kKStages], (uint32_t)((j + 2) / kKStages) & 1u, &sh.abort);
              wait_phase(&sh.s_free[j & 1], (uint32_t)(j >> 1) & 1u, &sh.abort);
            }
            tc_fence_after();
            if (leader) scores(j + 2, i * 6, i * 6 + 6);
            __syncwarp();
          }
        }
      }
      // nothing of this warp's is under way when the tensor memory is freed
      if (leader) umma_commit(&sh.idle);
      __syncwarp();
      mbar_wait(&sh.idle, 0u);
    } else if (warp == 11) {
      // ---- V rows of the blocks that reach behind the context. After the ring's first turn the
      // MMA warp, which has seen every block before, says when one is there: a parity alone
      // would also match an earlier turn. (The wait on v_full orders the copy before the reads.)
      for (int n = max(0, draft0); n < nb; ++n) {
        const int s = n % kVStages;
        if (n >= kVStages && !wait_phase(&sh.v_here[n - draft0], 0u, &sh.abort)) break;
        if (!wait_phase(&sh.v_full[s], (uint32_t)(n / kVStages) & 1u, &sh.abort)) break;
        for (int row = lane; row < kTcBlock; row += 32) {
          const int slot = (blk0 + n) * kTcBlock + row;
          if (slot < T0) continue;
#pragma unroll 1
          for (int c = 0; c < HD / 8; ++c) {
            uint4* at = reinterpret_cast<uint4*>(sV + s * T::kV + (c / 8) * T::kVBox + row * 128 + (((c & 7) ^ (row & 7)) << 4));
            if (slot >= slots) {
              *at = make_uint4(0, 0, 0, 0);
              continue;
            }
            uint4 v = *at;
            uint32_t hit = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t& u = e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w;
              const uint32_t lo = (u & 0x7f80u) == 0x7f80u, hi = (u & 0x7f800000u) == 0x7f800000u;
              if (lo) u &= 0xffff0000u;
              if (hi) u &= 0x0000ffffu;
              hit |= lo | hi;
            }
            if (hit) {
              *at = v;
              atomicOr(&sh.bad[n - draft0], 1);
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(&sh.v_ok[n - draft0]);
      }
    }
    __syncwarp();
  } else {
    // ---- softmax: group w, one row per thread
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int w = warp >> 2, row = tid & 127;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    float o[HD], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int d = 0; d < HD; ++d) o[d] = 0.f;
    for (int j = 0; 2 * j + w < nb; ++j) {
      const int n = 2 * j + w;
      const bool drafted = n >= draft0;
      wait_phase(&sh.s_full[j & 1], (uint32_t)(j >> 1) & 1u, &sh.abort);
      tc_fence_after();
      uint32_t u0[32], u1[32];
      tmem_ld32(lanes + (uint32_t)(j & 1) * kPair + (uint32_t)w * 64, u0);
      tmem_ld32(lanes + (uint32_t)(j & 1) * kPair + (uint32_t)w * 64 + 32, u1);
      tmem_ld_wait();
      tc_fence_before();
      mbar_arrive(&sh.s_free[j & 1]);
      const unsigned long long see = drafted ? ta_sees(anc, (blk0 + n) * kTcBlock - T0) : ~0ull;
      const float f = ta_softmax_block(u0, u1, drafted, see, m, l, lanes + T::kP + (uint32_t)w * 96);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&sh.p_ready[w]);
#pragma unroll
      for (int h = 0; h < T::BOX; ++h) {
        wait_phase(&sh.o_full[w], (uint32_t)(j * T::BOX + h) & 1u, &sh.abort);
        tc_fence_after();
        tmem_ld32(lanes + T::kO, u0);
        tmem_ld32(lanes + T::kO + 32u, u1);
        tmem_ld_wait();
        tc_fence_before();
        mbar_arrive(&sh.o_free[w]);
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          o[h * 64 + e] = fmaf(o[h * 64 + e], f, __uint_as_float(u0[e]));
          o[h * 64 + 32 + e] = fmaf(o[h * 64 + 32 + e], f, __uint_as_float(u1[e]));
        }
      }
      if (drafted) {
        // values that were taken out of V, added where they are seen
        wait_phase(&sh.v_ok[n - draft0], 0u, &sh.abort);
        if (sh.bad[n - draft0]) ta_add_nonfinite<__nv_bfloat16, HD>(P, k, o, see, (blk0 + n) * kTcBlock, T0);
      }
    }
    // every MMA has completed (this group waited for its last O, and so did the other)
    asm volatile("bar.sync 1, 256;" ::: "memory");
    float* sO = reinterpret_cast<float*>(base);
    float* sML = sO + 2 * kTcRows * (HD + 4);
    float* mine = sO + (w * kTcRows + row) * (HD + 4);
#pragma unroll
    for (int d = 0; d < HD; d += 4) *reinterpret_cast<float4*>(mine + d) = make_float4(o[d], o[d + 1], o[d + 2], o[d + 3]);
    sML[(w * kTcRows + row) * 2] = m, sML[(w * kTcRows + row) * 2 + 1] = l;
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (!sh.abort) ta_finish<HD, 2, kTcRows, 256>(P, k, sO, sML, tid);
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && sh.abort) atomicExch(a.err, kErrTreeWait);
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
  }
}

}  // namespace

cudaError_t configure_tree_attn_tc() {
  cudaError_t e = cudaFuncSetAttribute(tree_attn_tc_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcTile<64>::kSmem);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(tree_attn_tc_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcTile<128>::kSmem);
  return e;
}

cudaError_t launch_tree_attn_tc(const TAKernelArgs& P, int hd, dim3 grid, cudaStream_t st) {
  const CUtensorMap &mk = *static_cast<const CUtensorMap*>(P.a.tc_k), &mv = *static_cast<const CUtensorMap*>(P.a.tc_v);
  if (hd == 64)
    tree_attn_tc_kernel<64><<<grid, kTcAttnThreads, TcTile<64>::kSmem, st>>>(P, mk, mv);
  else
    tree_attn_tc_kernel<128><<<grid, kTcAttnThreads, TcTile<128>::kSmem, st>>>(P, mk, mv);
  return cudaGetLastError();
}

}  // namespace dllm
