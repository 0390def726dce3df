// tree_kv.cu — the cache rows of drafted tokens: append a tree's K/V rows behind
// the cached context, and move the rows of an accepted path to the front of them.
// Both are copies, bound by memory (and, at small sizes, by the launch).
#include "kernels.cuh"
#include "verify.cuh"

namespace dllm {
namespace {

template <typename T>
DLLM_DEV void put4(T* p, float4 f);
template <>
DLLM_DEV void put4<float>(float* p, float4 f) {
  *reinterpret_cast<float4*>(p) = f;
}
template <>
DLLM_DEV void put4<__nv_bfloat16>(__nv_bfloat16* p, float4 f) {  // the cache's own rounding: to nearest, ties to even
  __nv_bfloat162 a = __floats2bfloat162_rn(f.x, f.y), b = __floats2bfloat162_rn(f.z, f.w);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
}

// Thread per 4 dims of a K or V row. Grid (row chunks, sequences).
template <typename KT>
__global__ void __launch_bounds__(256)
    tree_append_kernel(const TreeSeq* seqs, const __grid_constant__ TreeT0 t0, KvLayout kv, const float* k,
                       const float* v, KT* kc, KT* vc, int kvh, int hd, int* err) {
  const TreeSeq s = seqs[blockIdx.y];
  const int per = kvh * hd / 4;
  const int total = s.m * per;
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < total; i += gridDim.x * blockDim.x) {
    const int node = i / per, e = (i - node * per) * 4;
    const int head = e / hd, d = e - head * hd;
    const int slot = t0.t0[blockIdx.y] + node;
    if (slot < 0 || slot >= kv.max_slots || s.seq >= kv.num_seqs) {
      atomicExch(err, kErrKvRange);  // checked by the host; kept so that no argument can make the store stray
      continue;
    }
    const size_t src = (size_t)(s.row0 + node) * kvh * hd + e;
    const long long dst = kv.offset(s.seq, slot, head) + d;
    put4(kc + dst, *reinterpret_cast<const float4*>(k + src));
    put4(vc + dst, *reinterpret_cast<const float4*>(v + src));
  }
}

// Thread per 16-byte column of one (sequence, layer, K or V, head): it carries the
// column through the accepted rows in order, kBatch loads ahead of their stores.
// path is strictly increasing with path[j] >= j, so a row is never stored over
// before it was loaded: the rows still to load lie behind path[j + kBatch - 1] >=
// j + kBatch - 1, the last row stored.
constexpr int kBatch = 8;

__global__ void __launch_bounds__(256)
    tree_commit_kernel(const __grid_constant__ CommitArgs a, KvLayout kv, char* kpool, char* vpool, size_t layer_bytes,
                       int layers, int esize, int kvh, int cols) {
  __shared__ long long off[2][kTreeMaxNodes];  // element offsets of head 0: sources, targets
  const int s = blockIdx.y;
  const int first = a.first[s], len = a.len[s], t0 = a.t0[s];
  for (int j = first + threadIdx.x; j < len; j += blockDim.x) {
    off[0][j] = kv.offset(a.seq[s], t0 + a.path[s][j], 0);
    off[1][j] = kv.offset(a.seq[s], t0 + j, 0);
  }
  __syncthreads();
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= layers * 2 * kvh * cols) return;
  const int col = i % cols, head = (i / cols) % kvh, which = (i / (cols * kvh)) & 1, layer = i / (2 * cols * kvh);
  char* base = (which ? vpool : kpool) + (size_t)layer * layer_bytes + (size_t)head * kv.head_stride * esize + col * 16;
  for (int j = first; j < len; j += kBatch) {
    uint4 r[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (j + u < len) r[u] = *reinterpret_cast<const uint4*>(base + off[0][j + u] * esize);
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (j + u < len) *reinterpret_cast<uint4*>(base + off[1][j + u] * esize) = r[u];
  }
}

}  // namespace

cudaError_t op_tree_append(const TreeSeq* seqs, int n_seqs, int max_m, const TreeT0& t0, const KvLayout& kv,
                           const float* k, const float* v, void* kc, void* vc, int kv_dtype, int kvh, int hd, int* err,
                           cudaStream_t st) {
  const dim3 grid((unsigned)((max_m * kvh * hd / 4 + 255) / 256), n_seqs);
  if (kv_dtype == 0)
    tree_append_kernel<float><<<grid, 256, 0, st>>>(seqs, t0, kv, k, v, (float*)kc, (float*)vc, kvh, hd, err);
  else
    tree_append_kernel<__nv_bfloat16>
        <<<grid, 256, 0, st>>>(seqs, t0, kv, k, v, (__nv_bfloat16*)kc, (__nv_bfloat16*)vc, kvh, hd, err);
  return cudaGetLastError();
}

cudaError_t op_tree_commit(const CommitArgs& a, const KvLayout& kv, void* kpool, void* vpool, size_t layer_elems,
                           int layers, int kv_dtype, int kvh, int hd, cudaStream_t st) {
  const int esize = kv_dtype == 0 ? 4 : 2, cols = hd * esize / 16;
  const dim3 grid((unsigned)((layers * 2 * kvh * cols + 255) / 256), a.n_seqs);
  tree_commit_kernel<<<grid, 256, 0, st>>>(a, kv, (char*)kpool, (char*)vpool, layer_elems * esize, layers, esize, kvh,
                                           cols);
  return cudaGetLastError();
}

}  // namespace dllm
