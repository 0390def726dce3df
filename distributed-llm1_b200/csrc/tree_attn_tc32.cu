// tree_attn_tc32.cu — tree attention over an fp32 cache on the tcgen05 tensor cores.
//
// The tensor cores have no fp32 operands, so K and V are cut like q and p, into three bf16
// terms, by truncation: 8 + 8 + 8 bits, which is every bit of an fp32 value. Of the nine
// products of two such sums the six largest are kept (what is left out is below 2^-23 of
// the product), and they run smallest first into one accumulator.
//
// One CTA, four warpgroups, one 128-row tile over its share of the 64-slot blocks:
//   producer (1 warp)    TMA: halves of 32 slots of K and V, as they lie, into two buffers
//   converters (4 warps) a half from a buffer into the three planes of a K or V operand;
//                        rows behind the last node become zero, and non-finite values of
//                        drafted rows are taken out of V (see ta_add_nonfinite)
//   MMA (1 warp)         S(n + 1) = q K^T, then O(n) = P V
//   two softmax groups   as in tree_attn_tc.cu; group w takes the blocks n % 2 = w
// The planes of K and of V are single: K(n + 1) is converted while O(n - 1) runs, V(n)
// while S(n + 1) runs. Tensor memory: S 2 x 64, P 2 x 96, O 128 columns.
// Bound: per block 48 MMAs of 128 x 64 x 16 (49 cycles) and 24 of 128 x 128 x 16 (65): 3900
// cycles, 2.0 us, against 1.5 us for 64 slots x 1024 bytes at one SM's share of HBM. Measured
// with clock stamps, 8 sequences x 7 nodes x 6 heads, six blocks per CTA, cold cache: 6050 cycles
// per block between the first S and the last O, 10 400 until the first S and 8700 from the last O
// to the end (66, 19 and 15 % of the kernel). In the loop the MMAs, the converters and the copies
// share 128 bytes of shared memory per cycle, and V(n) waits for O(n - 1) before it is
// converted. The upper terms of q in tensor memory with two sets of K planes made a block 8 %
// shorter but cost as much at the start; several loads per converter thread in flight only held the MMAs up
// (64 nodes x 7 heads at 32000 slots: 221 us one at a time, 241 two). The mma.sync kernel with
// tf32 terms takes 16000 cycles per block for 64 rows. 112 bytes are spilled at HD = 128.
#include "tree_attn_tc.cuh"

namespace dllm {
namespace {

constexpr int kTc32Threads = 512;
constexpr int kHalf = kTcBlock / 2;  // slots per staged copy

template <int HD>
struct Tc32Tile {
  static constexpr int BOX = HD / 64;
  static constexpr int kQPlane = BOX * kTcRows * 128;
  static constexpr int kBox = kTcBlock * 128;          // bytes of 64 slots x 64 dims, bf16
  static constexpr int kPlane = BOX * kBox;            // one term of a K or V block
  static constexpr int kStage = kHalf * HD * 4;        // 32 slots, fp32
  static constexpr int kOut = 2 * kTcRows * (HD + 6) * 4;
  static constexpr int kSmem = 1024 + 3 * kQPlane + 6 * kPlane + 2 * kStage;
  static_assert(kOut <= 3 * kQPlane + 6 * kPlane, "results reuse the operands' memory");
  static_assert(kSmem + 512 <= 227 * 1024, "shared memory");
  static constexpr uint32_t kP = 128, kO = 320;
};

struct Tc32Shared {
  uint64_t in_full[2], in_empty[2];            // staged halves
  uint64_t k_ready, k_free, v_ready, v_free;   // the converted planes
  uint64_t s_full[2], p_ready[2], o_full[2], o_free[2];
  uint64_t v_ok[2];                            // the (at most two) blocks with drafted rows
  uint64_t idle;
  uint32_t tmem;
  int bad[2];
  volatile int abort;
};

// 8 fp32 values -> three times 8 bf16, truncated: 8 bits each, 24 in all.
DLLM_DEV void cut3(const float4& a, const float4& b, uint4& h, uint4& m, uint4& l) {
  const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t hh[4], mm[4], ll[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float x = v[2 * e], y = v[2 * e + 1];
    hh[e] = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
    x -= __uint_as_float(__float_as_uint(x) & 0xffff0000u), y -= __uint_as_float(__float_as_uint(y) & 0xffff0000u);
    mm[e] = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
    x -= __uint_as_float(__float_as_uint(x) & 0xffff0000u), y -= __uint_as_float(__float_as_uint(y) & 0xffff0000u);
    ll[e] = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
  }
  h = make_uint4(hh[0], hh[1], hh[2], hh[3]);
  m = make_uint4(mm[0], mm[1], mm[2], mm[3]);
  l = make_uint4(ll[0], ll[1], ll[2], ll[3]);
}

// Products (term of q or p, term of K or V), smallest first: (2,0) (1,1) (0,2) (1,0) (0,1)
// (0,0); term 0 is the highest.
constexpr int kProducts = 6;
DLLM_DEV uint32_t term_a(int i) { return 0x001012u >> (4 * i) & 3u; }
DLLM_DEV uint32_t term_b(int i) { return 0x010210u >> (4 * i) & 3u; }

template <int HD>
__global__ void __launch_bounds__(kTc32Threads, 1)
    tree_attn_tc32_kernel(const __grid_constant__ TAKernelArgs P, const __grid_constant__ CUtensorMap tmK,
                          const __grid_constant__ CUtensorMap tmV) {
  using T = Tc32Tile<HD>;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) Tc32Shared sh;
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
  const int draft0 = T0 / kTcBlock - blk0;  // the first block (of this CTA's) with drafted rows

  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* sQ = base;
  unsigned char* sK = base + 3 * T::kQPlane;
  unsigned char* sV = sK + 3 * T::kPlane;
  unsigned char* sIn = sV + 3 * T::kPlane;

  if (tid == 0) {
    for (int w = 0; w < 2; ++w) {
      mbar_init(&sh.in_full[w], 1), mbar_init(&sh.in_empty[w], 128);
      mbar_init(&sh.s_full[w], 1), mbar_init(&sh.p_ready[w], 128);
      mbar_init(&sh.o_full[w], 1), mbar_init(&sh.o_free[w], 128);
      mbar_init(&sh.v_ok[w], 128);
      sh.bad[w] = 0;
    }
    mbar_init(&sh.k_ready, 128), mbar_init(&sh.k_free, 1), mbar_init(&sh.v_ready, 128), mbar_init(&sh.v_free, 1);
    mbar_init(&sh.idle, 1);
    sh.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
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
  if (warp < 8 || warp == 9) {  // the softmax groups bring q, the MMA warp waits for it
    if (warp < 8) ta_load_q<HD, 256>(P, k, sQ, tid);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // q is read by the MMA
    asm volatile("bar.sync 2, 288;" ::: "memory");
  }

  // Tiles in the order of conversion: K(0), then K(n + 1) and V(n) for each n; every tile in
  // two halves. Calls f(is_v, block, half, running number of the half).
  auto tiles = [&](auto f) {
    int i = 0;
    bool ok = f(false, 0, 0, 0) && f(false, 0, 1, 1);
    i = 2;
    for (int n = 0; ok && n < nb; ++n) {
      if (n + 1 < nb) {
        ok = f(false, n + 1, 0, i) && f(false, n + 1, 1, i + 1);
        i += 2;
      }
      if (ok) ok = f(true, n, 0, i) && f(true, n, 1, i + 1);
      i += 2;
    }
  };

  if (warp >= 8 && warp < 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 8 && lane == 0) {
      // ---- producer. The pools are one tensor of rows (layer, page, head, slot); a page holds at
      // least 32 slots, so a half lies in one page. Halves behind the end are loaded again.
      const int page = 1 << a.kv.log2_page;
      int sent = 0;
      tiles([&](bool is_v, int n, int h, int i) {
        const int slot = min((blk0 + n) * kTcBlock + h * kHalf, slots - 1) & ~(kHalf - 1);
        const int row = a.tc_row0 +
                        (a.kv.page_table[(size_t)k.sq.seq * a.kv.max_pages + (slot >> a.kv.log2_page)] * a.kvh + k.head) * page +
                        (slot & (page - 1));
        if (!wait_phase(&sh.in_empty[i & 1], ((uint32_t)(i >> 1) & 1u) ^ 1u, &sh.abort)) return false;
        mbar_expect_tx(&sh.in_full[i & 1], T::kStage);
        tma_load_2d(sIn + (i & 1) * T::kStage, is_v ? &tmV : &tmK, 0, row, &sh.in_full[i & 1]);
        sent = i + 1;
        return true;
      });
      // whatever happened to the others, the copies under way land before the CTA ends
      for (int i = max(0, sent - 2); i < sent; ++i) mbar_wait(&sh.in_full[i & 1], (uint32_t)(i >> 1) & 1u);
    } else if (warp == 9) {
      // ---- MMA issuer: the whole warp runs the loop, one elected lane issues (see tree_attn_tc.cu)
      const uint32_t leader = elect_one();
      const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kTcRows >> 4) << 24);  // fp32 += bf16 x bf16
      const uint32_t id_s = idesc | ((uint32_t)(kTcBlock >> 3) << 17);         // N = 64 slots, K-major
      const uint32_t id_o = idesc | ((uint32_t)(HD >> 3) << 17) | (1u << 16);  // N = hd, B with N contiguous
      auto scores = [&](int n) {
        wait_phase(&sh.k_ready, (uint32_t)n & 1u, &sh.abort);
        tc_fence_after();
        if (leader) {
#pragma unroll 1
          for (int i = 0; i < kProducts; ++i)
#pragma unroll
            for (int x = 0; x < T::BOX; ++x) {
              const uint64_t ad = umma_desc_sw128(sQ + term_a(i) * T::kQPlane + x * (kTcRows * 128));
              const uint64_t bd = umma_desc_sw128(sK + term_b(i) * T::kPlane + x * T::kBox);
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                umma_bf16(tmem + (uint32_t)(n & 1) * 64, ad + 2ull * kk, bd + 2ull * kk, id_s, (uint32_t)(i || x || kk));
            }
          umma_commit(&sh.k_free);
          umma_commit(&sh.s_full[n & 1]);
        }
        __syncwarp();
      };
      scores(0);
      for (int n = 0; n < nb; ++n) {
        if (n + 1 < nb) scores(n + 1);  // S is free: this warp has waited for P(n - 1)
        const int w = n & 1;
        wait_phase(&sh.v_ready, (uint32_t)n & 1u, &sh.abort);
        wait_phase(&sh.p_ready[w], (uint32_t)(n >> 1) & 1u, &sh.abort);
        if (n > 0) wait_phase(&sh.o_free[w ^ 1], (uint32_t)((n - 1) >> 1) & 1u, &sh.abort);
        tc_fence_after();
        if (leader) {
#pragma unroll 1
          for (int i = 0; i < kProducts; ++i) {
            const uint32_t ap = tmem + T::kP + (uint32_t)w * 96 + term_a(i) * 32;
            const uint64_t bd = umma_desc_mn_sw128(sV + term_b(i) * T::kPlane, T::kBox);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)  // 16 slots: 2048 bytes on
              umma_bf16_ts(tmem + T::kO, ap + 8u * kk, bd + 128ull * kk, id_o, (uint32_t)(i || kk));
          }
          umma_commit(&sh.v_free);
          umma_commit(&sh.o_full[w]);
        }
        __syncwarp();
      }
      // nothing of this warp's is under way when the tensor memory is freed
      if (leader) umma_commit(&sh.idle);
      __syncwarp();
      mbar_wait(&sh.idle, 0u);
    }
    __syncwarp();
  } else if (warp >= 12) {
    // ---- converters
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    const int me = tid - 384;
    tiles([&](bool is_v, int n, int h, int i) {
      if (!wait_phase(&sh.in_full[i & 1], (uint32_t)(i >> 1) & 1u, &sh.abort)) return false;
      // the planes of the block before have been read
      if (h == 0 && n > 0 && !wait_phase(is_v ? &sh.v_free : &sh.k_free, (uint32_t)(n - 1) & 1u, &sh.abort)) return false;
      const unsigned char* in = sIn + (i & 1) * T::kStage;
      unsigned char* out = is_v ? sV : sK;
      const int slot0 = (blk0 + n) * kTcBlock + h * kHalf;
      const bool edge = is_v && slot0 + kHalf > T0;  // rows that some nodes do not see
#pragma unroll 1
      for (int j = me; j < kHalf * HD / 8; j += 128) {
        const int s = j / (HD / 8), c = j % (HD / 8), row = h * kHalf + s;
        // lanes 4-7 of each eight read their second half first: the eight cover every bank
        const int swap = (me & 4) << 2;
        float4 f = *reinterpret_cast<const float4*>(in + j * 32 + swap), g = *reinterpret_cast<const float4*>(in + j * 32 + (swap ^ 16));
        if (swap) {
          const float4 z = f;
          f = g, g = z;
        }
        if (edge && slot0 + s >= T0) {
          if (slot0 + s >= slots) {
            f = g = make_float4(0.f, 0.f, 0.f, 0.f);
          } else {
            bool hit = false;
            auto clean = [&](float& v) {
              if (!is_finite(v)) v = 0.f, hit = true;
            };
            clean(f.x), clean(f.y), clean(f.z), clean(f.w), clean(g.x), clean(g.y), clean(g.z), clean(g.w);
            if (hit) atomicOr(&sh.bad[n - draft0], 1);
          }
        }
        uint4 hi, mi, lo;
        cut3(f, g, hi, mi, lo);
        unsigned char* at = out + (c / 8) * T::kBox + row * 128 + (((c & 7) ^ (row & 7)) << 4);
        *reinterpret_cast<uint4*>(at) = hi;
        *reinterpret_cast<uint4*>(at + T::kPlane) = mi;
        *reinterpret_cast<uint4*>(at + 2 * T::kPlane) = lo;
      }
      mbar_arrive(&sh.in_empty[i & 1]);
      if (h == 1) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(is_v ? &sh.v_ready : &sh.k_ready);
        if (is_v && n >= draft0) mbar_arrive(&sh.v_ok[n - draft0]);
      }
      return true;
    });
    __syncwarp();
  } else {
    // ---- softmax: group w, one row per thread
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int w = warp >> 2, row = tid & 127;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    float o[HD], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int d = 0; d < HD; ++d) o[d] = 0.f;
    for (int n = w; n < nb; n += 2) {
      const uint32_t ph = (uint32_t)(n >> 1) & 1u;
      const bool drafted = n >= draft0;
      wait_phase(&sh.s_full[w], ph, &sh.abort);
      tc_fence_after();
      uint32_t u0[32], u1[32];
      tmem_ld32(lanes + (uint32_t)w * 64, u0);
      tmem_ld32(lanes + (uint32_t)w * 64 + 32, u1);
      tmem_ld_wait();
      const unsigned long long see = drafted ? ta_sees(anc, (blk0 + n) * kTcBlock - T0) : ~0ull;
      const float f = ta_softmax_block(u0, u1, drafted, see, m, l, lanes + T::kP + (uint32_t)w * 96);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&sh.p_ready[w]);
      wait_phase(&sh.o_full[w], ph, &sh.abort);
      tc_fence_after();
#pragma unroll
      for (int d = 0; d < HD; d += 32) {
        tmem_ld32(lanes + T::kO + (uint32_t)d, u0);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e) o[d + e] = fmaf(o[d + e], f, __uint_as_float(u0[e]));
      }
      tc_fence_before();
      mbar_arrive(&sh.o_free[w]);
      if (drafted) {
        wait_phase(&sh.v_ok[n - draft0], 0u, &sh.abort);
        if (sh.bad[n - draft0]) ta_add_nonfinite<float, HD>(P, k, o, see, (blk0 + n) * kTcBlock, T0);
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

cudaError_t configure_tree_attn_tc32() {
  cudaError_t e = cudaFuncSetAttribute(tree_attn_tc32_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tc32Tile<64>::kSmem);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(tree_attn_tc32_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tc32Tile<128>::kSmem);
  return e;
}

cudaError_t launch_tree_attn_tc32(const TAKernelArgs& P, int hd, dim3 grid, cudaStream_t st) {
  const CUtensorMap &mk = *static_cast<const CUtensorMap*>(P.a.tc_k), &mv = *static_cast<const CUtensorMap*>(P.a.tc_v);
  if (hd == 64)
    tree_attn_tc32_kernel<64><<<grid, kTc32Threads, Tc32Tile<64>::kSmem, st>>>(P, mk, mv);
  else
    tree_attn_tc32_kernel<128><<<grid, kTc32Threads, Tc32Tile<128>::kSmem, st>>>(P, mk, mv);
  return cudaGetLastError();
}

}  // namespace dllm
