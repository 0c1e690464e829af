// Losses over the vocabulary (include/pe_vocab.h): next-token cross entropy and distillation from a teacher's
// top logits, forward, backward, and both from one read of the logits.
//
// With m = max z, s = sum exp(z - m) and s_T = sum exp((z - m) / T) of a row,
//     hard = (m - z_y) + ln s
//     soft = T^2 sum_k p_k (ln p_k + (m - z_k) / T + ln s_T)
//     dz_j = c (hw e^(z_j - m) / s + sw T P e^((z_j - m) / T) / s_T),  P = sum_k p_k (1, or 0 with no pair present)
// and at the at most K + 1 places that the label and the teacher name, dz_j less c hw [j = y] and
// c sw T sum_{k: id_k = j} p_k.  A workgroup takes a row; those few places are written again behind the dense
// ones, by one thread for each different id.
//
// Bound by memory: one read of the logits forward, one read and one write backward, and one of each in the step, whose
// workgroup holds its row in registers.  Rows are read in 16-byte pieces from the first 16-byte address on; the up
// to seven elements on either side of the pieces are a thread's each.
#include "pe_common.h"
#include "pe_internal.h"
#include "pe_vocab.h"

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

// the row's label; false when the row does not count.  Without labels every row counts, with label -1
__device__ __forceinline__ bool row_label(const LossArgs& a, int64_t r, int64_t& y) {
  y = -1;
  if (!a.labels) return true;
  if (a.shift) {
    if (r % a.shift == a.shift - 1) return false;
    r += 1;
  }
  y = load_id(a.labels, a.label_bytes, r);
  return y != a.ignore;
}

// 2^x in one instruction; results below 2^-126 are 0
__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

// 16 bytes of a row as floats
template <int DT> struct Vec {
  static constexpr int ES = DT == 1 ? 4 : 2, N = 16 / ES;
  static __device__ __forceinline__ void unpack(const u32x4& r, float (&x)[N]) {
    if constexpr (DT == 0) unpack8(r, x);
    else if constexpr (DT == 2) unpack8_h(r, x);
    else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = r[i];  // a bit cast of the vector's element itself reads element 0
        x[i] = __builtin_bit_cast(float, w);
      }
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float (&x)[N]) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == 1) r[i] = __builtin_bit_cast(uint32_t, x[i]);
      else r[i] = pack2<DT>(x[2 * i], x[2 * i + 1]);
    }
    return r;
  }
};

// A row of V elements at `p`: `head` single elements, `nvec` pieces of 16 bytes, and single elements to the end.
// single(t) is the single element of thread t, or -1.
template <int DT> struct Row {
  const char* p;
  int V, head, nvec;
  __device__ __forceinline__ Row(const char* q, int v) : p(q), V(v) {
    constexpr int ES = Vec<DT>::ES;
    head = min((int)((16 - ((uintptr_t)p & 15)) & 15) / ES, V);
    nvec = (V - head) / Vec<DT>::N;
  }
  __device__ __forceinline__ int single(int t) const {
    const int j = t < head ? t : t + nvec * Vec<DT>::N;
    return j < V ? j : -1;
  }
  __device__ __forceinline__ int first(int k) const { return head + k * Vec<DT>::N; }  // element of piece k
  __device__ __forceinline__ u32x4 load(int k) const { return *(const u32x4*)(p + (int64_t)first(k) * Vec<DT>::ES); }
};
// the pieces of a row whose gradient is 16 bytes aligned where the row is, else element by element
template <int DT> __device__ __forceinline__ void store_piece(char* dz, int j, bool together, const float (&x)[Vec<DT>::N]) {
  if (together) {
    *(u32x4*)(dz + (int64_t)j * Vec<DT>::ES) = Vec<DT>::pack(x);
  } else {
#pragma unroll
    for (int e = 0; e < Vec<DT>::N; ++e) put<DT>(dz, j + e, x[e]);
  }
}

// a maximum and the sums of exponentials relative to it; -inf and no sums to begin with.  A maximum of -inf is no
// reference (its differences would be NaN): 0 is taken then, relative to which its exponentials are 0 as well
struct Stat { float m, s, t; };
__device__ __forceinline__ float reference(float m) { return m == -INFINITY ? 0.f : m; }

template <bool HARD, bool SOFT> __device__ __forceinline__ void rescale(Stat& x, float m, float lt) {
  const float d = x.m - reference(m);
  if (HARD) x.s *= ex2(d * LOG2E);
  if (SOFT) x.t *= ex2(d * lt);
  x.m = m;
}
template <bool HARD, bool SOFT, int N> __device__ __forceinline__ void add(Stat& st, const float (&x)[N], float lt) {
  const float ref = reference(st.m);
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float d = x[e] - ref;
    if (HARD) st.s += ex2(d * LOG2E);
    if (SOFT) st.t += ex2(d * lt);
  }
}
template <bool HARD, bool SOFT> __device__ __forceinline__ Stat join(Stat x, Stat y, float lt) {
  const float m = fmaxf(x.m, y.m);
  rescale<HARD, SOFT>(x, m, lt);
  rescale<HARD, SOFT>(y, m, lt);
  return Stat{m, x.s + y.s, x.t + y.t};
}

template <int T> __device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = red[0];
  for (int i = 1; i < T / 64; ++i) r += red[i];
  return r;
}
template <int T> __device__ __forceinline__ float block_max(float v, float* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = red[0];
  for (int i = 1; i < T / 64; ++i) r = fmaxf(r, red[i]);
  return r;
}

}  // namespace

constexpr int U = 4;  // pieces a thread has in flight where the row is not held

// NC > 0: the row is held in registers, NC pieces a thread (the step, rows of up to NC T pieces); 0: it is read
// once for the sums (forward) or the gradient (backward), or for both in turn (the step of a longer row)
template <int DT, int PHASE, bool HARD, bool SOFT, int T, int NC>
__global__ __launch_bounds__(T) void loss_row_kernel(LossArgs a) {
  __shared__ float red[T / 64];
  __shared__ Stat wred[T / 64];
  __shared__ int32_t tid_l[SOFT ? PE_LOSS_MAX_TOP_K : 1];  // the teacher's ids, -1 where absent
  __shared__ float tp_l[SOFT ? PE_LOSS_MAX_TOP_K : 1];     // and probabilities
  using W = Vec<DT>;
  constexpr int N = W::N;
  const int64_t r = blockIdx.x;
  const int t = threadIdx.x, V = a.V;
  const char* z = (const char*)a.z + r * a.z_rs * W::ES;
  char* dz = PHASE == LOSS_FWD ? nullptr : (char*)a.dz + r * a.dz_rs * W::ES;
  const Row<DT> row(z, V);
  const int one = row.single(t);
  const bool together = (((uintptr_t)z ^ (uintptr_t)dz) & 15) == 0;
  int64_t y;
  if (!row_label(a, r, y)) {
    if (PHASE != LOSS_FWD) {
      const float zero[N] = {};
      for (int k = t; k < row.nvec; k += T) store_piece<DT>(dz, row.first(k), together, zero);
      if (one >= 0) put<DT>(dz, one, 0.f);
    }
    if (t == 0) {
      if (PHASE != LOSS_BWD) a.row_loss[r] = 0.f;
      if (PHASE == LOSS_FWD && a.stats) a.stats[3 * r] = a.stats[3 * r + 1] = a.stats[3 * r + 2] = 0.f;
    }
    return;
  }
  const bool bad = a.labels && (y < 0 || y >= V);
  const float lt = LOG2E / a.T;

  Stat st{-INFINITY, 0.f, 0.f};
  u32x4 held[NC > 0 ? NC : 1];
  const float xone = one >= 0 ? elem<DT>(z, one) : -INFINITY;
  if (PHASE == LOSS_BWD) {
    st = Stat{a.stats[3 * r], a.stats[3 * r + 1], a.stats[3 * r + 2]};
  } else if (NC > 0) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (c * T + t < row.nvec) held[c] = row.load(c * T + t);
    float mx = xone;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (c * T + t < row.nvec) {
        float x[N];
        W::unpack(held[c], x);
#pragma unroll
        for (int e = 0; e < N; ++e) mx = fmaxf(mx, x[e]);
      }
    }
    st.m = block_max<T>(mx, red);
    const float x1[1] = {xone};
    add<HARD, SOFT>(st, x1, lt);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (c * T + t < row.nvec) {
        float x[N];
        W::unpack(held[c], x);
        add<HARD, SOFT>(st, x, lt);
      }
    }
    if (HARD) st.s = block_sum<T>(st.s, red);
    if (SOFT) st.t = block_sum<T>(st.t, red);
  } else {
    const float x1[1] = {xone};
    st.m = xone;
    add<HARD, SOFT>(st, x1, lt);
    int k = t;
    for (; k + (U - 1) * T < row.nvec; k += U * T) {
      u32x4 raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = row.load(k + u * T);
      float x[U][N], mx = st.m;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        W::unpack(raw[u], x[u]);
#pragma unroll
        for (int e = 0; e < N; ++e) mx = fmaxf(mx, x[u][e]);
      }
      rescale<HARD, SOFT>(st, mx, lt);
#pragma unroll
      for (int u = 0; u < U; ++u) add<HARD, SOFT>(st, x[u], lt);
    }
    for (; k < row.nvec; k += T) {
      float x[N], mx = st.m;
      W::unpack(row.load(k), x);
#pragma unroll
      for (int e = 0; e < N; ++e) mx = fmaxf(mx, x[e]);
      rescale<HARD, SOFT>(st, mx, lt);
      add<HARD, SOFT>(st, x, lt);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
      st = join<HARD, SOFT>(st, Stat{__shfl_xor(st.m, o, 64), __shfl_xor(st.s, o, 64), __shfl_xor(st.t, o, 64)}, lt);
    if ((t & 63) == 0) wred[t >> 6] = st;
    __syncthreads();
    st = wred[0];
    for (int i = 1; i < T / 64; ++i) st = join<HARD, SOFT>(st, wred[i], lt);
  }
  if (PHASE == LOSS_FWD && a.stats && t == 0) {
    a.stats[3 * r] = st.m;
    a.stats[3 * r + 1] = st.s;
    a.stats[3 * r + 2] = st.t;
  }

  // the teacher's probabilities
  float P = 0.f;
  if (SOFT) {
    float mx = -INFINITY;
    for (int k = t; k < a.K; k += T) {
      const int64_t id = load_id(a.tid, a.tid_bytes, r * a.tid_rs + k);
      const float x = load_as_float(a.tlog, r * a.tlog_rs + k, a.tlog_dtype);
      const bool have = id >= 0 && id < V && x != -INFINITY;
      tid_l[k] = have ? (int32_t)id : -1;
      tp_l[k] = x;
      if (have) mx = fmaxf(mx, x);
    }
    mx = block_max<T>(mx, red);
    float n = 0.f;
    for (int k = t; k < a.K; k += T)
      if (tid_l[k] >= 0) n += ex2((tp_l[k] - mx) * lt);
    n = block_sum<T>(n, red);
    P = n != 0.f ? 1.f : 0.f;
    float sum = 0.f;
    for (int k = t; k < a.K; k += T) {
      float p = 0.f;
      if (tid_l[k] >= 0) {
        const float d = tp_l[k] - mx;
        p = ex2(d * lt) / n;
        if (PHASE != LOSS_BWD && p != 0.f)
          sum += p * ((d + st.m - elem<DT>(z, tid_l[k])) / a.T - logf(n) + logf(st.t));
      }
      tp_l[k] = p;
    }
    if (PHASE != LOSS_BWD) {
      sum = block_sum<T>(sum, red);
      P = n != 0.f ? 1.f : 0.f;
      if (t == 0) {
        float loss = a.sw * a.T * a.T * sum;
        if (HARD) loss += a.hw * (bad ? NAN : (st.m - elem<DT>(z, y)) + logf(st.s));
        a.row_loss[r] = bad ? NAN : loss;
      }
    }
    __syncthreads();
  } else if (PHASE != LOSS_BWD && t == 0) {
    a.row_loss[r] = bad ? NAN : a.hw * ((st.m - elem<DT>(z, y)) + logf(st.s));
  }

  if (PHASE == LOSS_FWD) return;
  float c = a.factor;
  if (a.dloss) c *= a.dloss[a.reduction == PE_LOSS_NONE ? r : 0];
  if (a.inv_count) c *= *a.inv_count;
  if (bad) c = NAN;
  const float ch = HARD ? c * a.hw / st.s : 0.f, ct = SOFT ? c * a.sw * a.T * P / st.t : 0.f;
  auto dense = [&](float x) {
    const float d = x - st.m;
    float g = 0.f;
    if (HARD) g = ch * ex2(d * LOG2E);
    if (SOFT) g = HARD ? g + ct * ex2(d * lt) : ct * ex2(d * lt);
    return g;
  };
  auto piece = [&](int k, const u32x4& raw) {
    float x[N];
    W::unpack(raw, x);
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = dense(x[e]);
    store_piece<DT>(dz, row.first(k), together, x);
  };
  if (one >= 0) put<DT>(dz, one, dense(xone));
  if (NC > 0) {
#pragma unroll
    for (int k = 0; k < NC; ++k)
      if (k * T + t < row.nvec) piece(k * T + t, held[k]);
  } else {
    int k = t;
    for (; k + (U - 1) * T < row.nvec; k += U * T) {
      u32x4 raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = row.load(k + u * T);
#pragma unroll
      for (int u = 0; u < U; ++u) piece(k + u * T, raw[u]);
    }
    for (; k < row.nvec; k += T) piece(k, row.load(k));
  }
  __syncthreads();
  // the named places again, by the first of the pairs with an id; the label's by thread 0 unless a pair has it
  if (SOFT) {
    for (int k = t; k < a.K; k += T) {
      const int32_t id = tid_l[k];
      if (id < 0) continue;
      float p = 0.f;
      bool first = true;
      for (int i = 0; i < a.K; ++i) {
        if (tid_l[i] == id) {
          first = first && i >= k;
          p += tp_l[i];
        }
      }
      if (!first) continue;
      float g = dense(elem<DT>(z, id)) - c * a.sw * a.T * p;
      if (HARD && id == y) g -= c * a.hw;
      put<DT>(dz, id, g);
    }
  }
  if (HARD && t == 0 && !bad) {
    bool named = false;
    if (SOFT)
      for (int i = 0; i < a.K; ++i) named |= tid_l[i] == y;
    if (!named) put<DT>(dz, y, dense(elem<DT>(z, y)) - c * a.hw);
  }
}

// 1 / rows that count, and the sum or mean of the row losses: one workgroup, thread t taking rows t, t + 1024, ...
template <bool SUM>
__global__ __launch_bounds__(1024) void loss_reduce_kernel(LossArgs a, float* loss, float* inv_count) {
  __shared__ double rs[16];
  __shared__ int32_t rn[16];
  const int t = threadIdx.x;
  double s = 0.;
  int32_t n = 0;
  for (int64_t r = t; r < a.rows; r += 1024) {
    int64_t y;
    if (SUM) s += a.row_loss[r];
    n += row_label(a, r, y) ? 1 : 0;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    if (SUM) s += __shfl_xor(s, o, 64);
    n += __shfl_xor(n, o, 64);
  }
  if ((t & 63) == 0) {
    rs[t >> 6] = s;
    rn[t >> 6] = n;
  }
  __syncthreads();
  if (t != 0) return;
  for (int i = 1; i < 16; ++i) {
    s += rs[i];
    n += rn[i];
  }
  if (SUM) *loss = (float)(a.reduction == PE_LOSS_MEAN ? s / (double)n : s);
  if (inv_count) *inv_count = 1.f / (float)n;
}

template <int DT, int PHASE, int T, int NC> static int run_loss(const LossArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)a.rows), block(T);
  if (a.sw == 0.f) hipLaunchKernelGGL((loss_row_kernel<DT, PHASE, true, false, T, NC>), grid, block, 0, s, a);
  else if (a.hw == 0.f) hipLaunchKernelGGL((loss_row_kernel<DT, PHASE, false, true, T, NC>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((loss_row_kernel<DT, PHASE, true, true, T, NC>), grid, block, 0, s, a);
  return hipGetLastError() == hipSuccess ? 0 : -7;
}

// Threads a row by its pieces: a wave for short rows, four for longer ones; the step the fewest registers that hold the
// row in a workgroup.
template <int DT, int PHASE> static int run_loss(const LossArgs& a, hipStream_t s) {
  const int pieces = a.V / Vec<DT>::N;
  if constexpr (PHASE == LOSS_STEP) {
    if (pieces <= 64 * 4) return run_loss<DT, PHASE, 64, 4>(a, s);
    if (pieces <= 256 * 4) return run_loss<DT, PHASE, 256, 4>(a, s);
    if (pieces <= 512 * 4) return run_loss<DT, PHASE, 512, 4>(a, s);
    if (pieces <= 512 * 8) return run_loss<DT, PHASE, 512, 8>(a, s);
    if (pieces <= 1024 * 8) return run_loss<DT, PHASE, 1024, 8>(a, s);
    if (pieces <= 1024 * 16) return run_loss<DT, PHASE, 1024, 16>(a, s);
    return run_loss<DT, PHASE, 1024, 0>(a, s);
  } else {
    if (pieces <= 64 * 4) return run_loss<DT, PHASE, 64, 0>(a, s);
    return run_loss<DT, PHASE, 256, 0>(a, s);
  }
}

template <int DT> static int loss_phase(int phase, const LossArgs& a, hipStream_t s) {
  if (phase == LOSS_FWD) return run_loss<DT, LOSS_FWD>(a, s);
  if (phase == LOSS_BWD) return run_loss<DT, LOSS_BWD>(a, s);
  return run_loss<DT, LOSS_STEP>(a, s);
}

int launch_loss(int dtype, int phase, const LossArgs& a, hipStream_t s) {
  if (a.rows == 0) return 0;
  if (dtype == 0) return loss_phase<0>(phase, a, s);
  if (dtype == 1) return loss_phase<1>(phase, a, s);
  return loss_phase<2>(phase, a, s);
}

int launch_loss_count(const LossArgs& a, float* inv_count, hipStream_t s) {
  hipLaunchKernelGGL(loss_reduce_kernel<false>, dim3(1), dim3(1024), 0, s, a, (float*)nullptr, inv_count);
  return hipGetLastError() == hipSuccess ? 0 : -7;
}

int launch_loss_reduce(const LossArgs& a, float* loss, float* inv_count, hipStream_t s) {
  hipLaunchKernelGGL(loss_reduce_kernel<true>, dim3(1), dim3(1024), 0, s, a, loss, inv_count);
  return hipGetLastError() == hipSuccess ? 0 : -7;
}

}  // namespace pe
