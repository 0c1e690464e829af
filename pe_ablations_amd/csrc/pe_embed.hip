// The scaled token embedding and its gradient (include/pe_vocab.h).
//
//     out[t] = weight[ids[t]] * scale        dweight[v] = scale * sum_{t: ids[t] = v} dy[t]
//
// Both are bound by memory.  The gradient sorts the tokens by id first (an int32 key and position each), then
// every row of the vocabulary finds its run of tokens by binary search and adds their rows in order, so each row
// of the gradient is written once, by one workgroup, and no sum depends on the order in which workgroups run.
#include "pe_common.h"
#include "pe_internal.h"

namespace pe {

namespace {

template <int DT> __device__ __forceinline__ float elem(const void* p, int64_t i) {
  if constexpr (DT == 1) return ((const float*)p)[i];
  else if constexpr (DT == 0) return bf2f(((const uint16_t*)p)[i]);
  else return h2f(((const uint16_t*)p)[i]);
}
template <int DT> __device__ __forceinline__ void put(void* p, int64_t i, float x) {
  if constexpr (DT == 1) ((float*)p)[i] = x;
  else if constexpr (DT == 0) ((uint16_t*)p)[i] = f2bf(x);
  else ((uint16_t*)p)[i] = f2h(x);
}

__device__ __forceinline__ int64_t load_id(const void* p, int bytes, int64_t i) {
  return bytes == 8 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

// x * s as an fp32 value: left to itself the compiler rounds the product of an fp16 store to fp16 at once
// (v_fma_mixlo_f16), which differs from torch's product and conversion in one place of a few hundred thousand
__device__ __forceinline__ float product(float x, float s) {
  float p = x * s;
  asm("" : "+v"(p));
  return p;
}

}  // namespace

template <int DT> __global__ __launch_bounds__(256) void embed_fwd_kernel(EmbedArgs a) {
  const int64_t row = blockIdx.x;
  const int64_t id = load_id(a.ids, a.id_bytes, row);
  const bool ok = id >= 0 && id < a.V;
  for (int j = threadIdx.x; j < a.H; j += 256)
    put<DT>(a.y, row * a.y_rs + j, ok ? product(elem<DT>(a.x, id * a.x_rs + j), a.scale) : NAN);
}

// The key of a token: its id, or V (behind every row of the vocabulary) when its gradient goes nowhere.
__device__ __forceinline__ int32_t token_key(const EmbedArgs& a, int64_t t) {
  const int64_t id = load_id(a.ids, a.id_bytes, t);
  return id < 0 || id >= a.V || id == a.pad ? (int32_t)a.V : (int32_t)id;
}

// A token's place in the sorted order is the number of tokens with a smaller key, or the same key and an earlier
// position.
__global__ __launch_bounds__(256) void embed_rank_kernel(EmbedArgs a) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  __shared__ int32_t tile[256];
  const int32_t key = t < a.n ? token_key(a, t) : 0;
  int32_t rank = 0;
  for (int64_t u0 = 0; u0 < a.n; u0 += 256) {
    __syncthreads();
    tile[threadIdx.x] = u0 + threadIdx.x < a.n ? token_key(a, u0 + threadIdx.x) : 0x7fffffff;
    __syncthreads();
    for (int i = 0; i < 256; ++i) rank += tile[i] < key || (tile[i] == key && u0 + i < t) ? 1 : 0;
  }
  if (t < a.n) {
    a.key[rank] = key;
    a.order[rank] = (int32_t)t;
  }
}

template <int DT> __global__ __launch_bounds__(256) void embed_bwd_kernel(EmbedArgs a) {
  const int32_t v = blockIdx.x;
  auto first = [&](int32_t key) {  // the first place with a key of at least `key`
    int64_t lo = 0, hi = a.n;
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      if (a.key[mid] < key) lo = mid + 1;
      else hi = mid;
    }
    return lo;
  };
  const int64_t i0 = first(v), i1 = first(v + 1);
  for (int j = threadIdx.x; j < a.H; j += 256) {
    float s = 0.f;
    for (int64_t i = i0; i < i1; ++i) s += elem<DT>(a.x, a.order[i] * a.x_rs + j);
    put<DT>(a.y, v * a.y_rs + j, product(s, a.scale));
  }
}

int launch_embed_fwd(int dtype, const EmbedArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)a.n), block(256);
  if (dtype == 0) hipLaunchKernelGGL(embed_fwd_kernel<0>, grid, block, 0, s, a);
  else if (dtype == 1) hipLaunchKernelGGL(embed_fwd_kernel<1>, grid, block, 0, s, a);
  else hipLaunchKernelGGL(embed_fwd_kernel<2>, grid, block, 0, s, a);
  return hipGetLastError() == hipSuccess ? 0 : -7;
}

int64_t embed_bwd_workspace(int64_t n, int64_t, int) { return 2 * ((n + 3) / 4 * 4) * 4 + 16; }

int launch_embed_bwd(int dtype, EmbedArgs a, void* ws, hipStream_t s) {
  a.key = (int32_t*)ws;
  a.order = a.key + (a.n + 3) / 4 * 4;
  if (a.n) {
    hipLaunchKernelGGL(embed_rank_kernel, dim3((unsigned)((a.n + 255) / 256)), dim3(256), 0, s, a);
    if (hipGetLastError() != hipSuccess) return -7;
  }
  const dim3 grid((unsigned)a.V), block(256);
  if (dtype == 0) hipLaunchKernelGGL(embed_bwd_kernel<0>, grid, block, 0, s, a);
  else if (dtype == 1) hipLaunchKernelGGL(embed_bwd_kernel<1>, grid, block, 0, s, a);
  else hipLaunchKernelGGL(embed_bwd_kernel<2>, grid, block, 0, s, a);
  return hipGetLastError() == hipSuccess ? 0 : -7;
}

}  // namespace pe
