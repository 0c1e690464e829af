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
// workgroup holds its row in registers (4096 x 50257 in bf16: forward 77 us, 5.3 TB/s, backward 138 us, 6.0 TB/s, step
// 164 us, 5.0 TB/s; 16384 x 50257 in fp32: forward alone 490 us, 6.7 TB/s).  Rows are read in 16-byte pieces from the
// first 16-byte address on; the up to seven elements on either side of the pieces are a thread's each.
#include <type_traits>

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
__device__ __forceinline__ bool row_label(const LossArgs& a, uint32_t r, int64_t& y) {
  y = -1;
  if (!a.labels) return true;
  if (a.shift) {
    r += 1;
    if (r % (uint32_t)a.shift == 0) return false;
  }
  y = load_id(a.labels, a.label_bytes, r);
  return y != a.ignore;
}

// What is summed.  At temperature 1 both parts have the same exponentials, at 2 the hard part's are the squares of
// the soft part's: one exponential an element in place of two.
enum { HARD = 1, SOFT = 2, BOTH = 3, BOTH_T1 = 4, BOTH_T2 = 5 };
constexpr bool has_hard(int mode) { return mode != SOFT; }
constexpr bool has_soft(int mode) { return mode != HARD; }

__device__ __forceinline__ float scalar(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
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
// single(t) is the single element of thread t, or -1.  A piece's place is an unsigned 32-bit offset from a base that
// is the same for every thread (rows below 4 GB), which takes one register where an address takes two.
template <int DT> struct Row {
  const char* body;
  int V, head, nvec;
  __device__ __forceinline__ Row(const char* p, int v) : V(v) {
    constexpr int ES = Vec<DT>::ES;
    head = min((int)((16 - ((uintptr_t)p & 15)) & 15) / ES, V);
    nvec = (V - head) / Vec<DT>::N;
    body = p + head * ES;
  }
  __device__ __forceinline__ int single(int t) const {
    const int j = t < head ? t : t + nvec * Vec<DT>::N;
    return j < V ? j : -1;
  }
  template <bool NT> __device__ __forceinline__ u32x4 load(int k) const {
    const u32x4* q = (const u32x4*)(body + (uint32_t)k * 16u);
    return NT ? __builtin_nontemporal_load(q) : *q;
  }
};
// piece k of the gradient's row, whose rows need not be aligned as the logits' are
template <int DT> __device__ __forceinline__ void store_piece(char* body, int k, bool stream, const float (&x)[Vec<DT>::N]) {
  u32x4_any* q = (u32x4_any*)(body + (uint32_t)k * 16u);
  const u32x4 r = Vec<DT>::pack(x);
  if (stream) {
    asm volatile("");  // on either side: else the compiler makes one plain store of the two
    __builtin_nontemporal_store((u32x4_any)r, q);
    asm volatile("");
  } else {
    *q = r;
  }
}

// a maximum and the sums of exponentials relative to it; -inf and no sums to begin with.  A maximum of -inf is no
// reference (its differences would be NaN): 0 is taken then, relative to which its exponentials are 0 as well
struct Stat { float m, s, t; };
__device__ __forceinline__ float reference(float m) { return m == -INFINITY ? 0.f : m; }

// the exponentials of an element d above (below 0) the maximum: of the hard part, and of the soft part
template <int MODE> __device__ __forceinline__ void exps(float d, float lt, float& e, float& et) {
  e = et = 0.f;
  if (MODE == BOTH_T2) {
    et = ex2(d * (0.5f * LOG2E));
    e = et * et;
  } else {
    if (has_hard(MODE)) e = ex2(d * LOG2E);
    if (MODE == SOFT || MODE == BOTH) et = ex2(d * lt);
  }
  if (MODE == BOTH_T1) et = e;
}
template <int MODE> __device__ __forceinline__ void rescale(Stat& x, float m, float lt) {
  float e, et;
  exps<MODE>(x.m - reference(m), lt, e, et);
  if (has_hard(MODE)) x.s *= e;
  if (has_soft(MODE)) x.t *= et;
  x.m = m;
}
template <int MODE, int N> __device__ __forceinline__ void add(Stat& st, const float (&x)[N], float lt) {
  const float ref = reference(st.m);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float e, et;
    exps<MODE>(x[i] - ref, lt, e, et);
    if (has_hard(MODE)) st.s += e;
    if (has_soft(MODE)) st.t += et;
  }
}
template <int MODE> __device__ __forceinline__ Stat join(Stat x, Stat y, float lt) {
  const float m = fmaxf(x.m, y.m);
  rescale<MODE>(x, m, lt);
  rescale<MODE>(y, m, lt);
  return Stat{m, x.s + y.s, x.t + y.t};
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}
template <int T> __device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = red[0];
#pragma unroll
  for (int i = 1; i < T / 64; ++i) r += red[i];
  return r;
}
template <int T> __device__ __forceinline__ float block_max(float v, float* red) {
  v = wave_max(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = red[0];
#pragma unroll
  for (int i = 1; i < T / 64; ++i) r = fmaxf(r, red[i]);
  return r;
}

}  // namespace

// Gradients beyond this size are stored past the 256 MB cache, smaller ones are left in it for the products that read
// them next (step, then both products of the output projection, hidden 512, vocabulary 32000: 62 MB 269 us streamed and
// 261 us not, 125 MB 424 and 432 us, 250 MB 695 and 704 us).
constexpr int64_t STREAM_BYTES = 96ll << 20;

constexpr int LOSS_ALONE = 3;  // a forward without a backward to follow: the logits are read past the caches

// NC > 0: the row is held in registers, NC pieces a thread (the step, rows of up to NC T pieces); 0: it is read
// once for the sums (forward) or the gradient (backward), or for both in turn (the step of a longer row), U pieces a
// thread in flight.
//
// The backward takes the rows last to first: those that the forward read last are still in the 256 MB cache behind
// the L2s, and a gradient that does not fit there is stored past it (4096 x 50257 in bf16, forward and backward:
// 244 us, 233 us with such stores, 214 us in reverse as well).
template <int DT, int PHASE, int MODE, int T, int NC, int U, int WPE = 1>
__global__ __launch_bounds__(T) __attribute__((amdgpu_waves_per_eu(WPE))) void loss_row_kernel(LossArgs a) {
  constexpr bool FWD = PHASE == LOSS_FWD || PHASE == LOSS_ALONE, BWD = PHASE == LOSS_BWD, NT = PHASE == LOSS_ALONE;
  __shared__ float red[2][T / 64];
  __shared__ Stat wred[T / 64];
  using W = Vec<DT>;
  constexpr int N = W::N;
  const int64_t r = BWD ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
  const int t = threadIdx.x, V = a.V;
  const char* z = (const char*)a.z + r * a.z_rs * W::ES;
  char* dz = FWD ? nullptr : (char*)a.dz + r * a.dz_rs * W::ES;
  const Row<DT> row(z, V);
  char* const dbody = FWD ? nullptr : dz + row.head * W::ES;
  const int one = row.single(t);
  int64_t y;
  if (!row_label(a, (uint32_t)r, y)) {
    if (!FWD) {
      const float zero[N] = {};
      for (int k = t; k < row.nvec; k += T) store_piece<DT>(dbody, k, a.stream, zero);
      if (one >= 0) put<DT>(dz, one, 0.f);
    }
    if (t == 0) {
      if (!BWD) a.row_loss[r] = 0.f;
      if (PHASE == LOSS_FWD) a.stats[3 * r] = a.stats[3 * r + 1] = a.stats[3 * r + 2] = 0.f;
    }
    return;
  }
  y = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(y >> 32)) << 32 |
                (uint32_t)__builtin_amdgcn_readfirstlane((int)y));
  const bool bad = a.labels && (y < 0 || y >= V);
  const float lt = LOG2E / a.T;

  Stat st{-INFINITY, 0.f, 0.f};
  // The named places, 64 of them or the label's alone, with their logits: fetched by the first wave beside the row and
  // left in LDS for its use at the end, before a held row's sums, where they made it spill, else behind the row
  __shared__ int32_t nid[64];
  __shared__ float np[64], nz[64];
  const int32_t* place = has_soft(MODE) ? a.place + r * (a.K + 1) : nullptr;
  const float* prob = has_soft(MODE) ? a.prob + r * (a.K + 1) : nullptr;
  int32_t id0 = -1;
  float p0 = 0.f;
  if (has_soft(MODE)) {
    if (t < 64 && t <= a.K) {
      id0 = place[t];
      p0 = prob[t];
    }
  } else if (t == 0 && !bad) {
    id0 = (int32_t)y;
  }
  u32x4 held[NC > 0 ? NC : 1];
  // between two uses of the held row: else the compiler keeps its elements as floats, twice the registers
  auto keep_packed = [&] {
#pragma unroll
    for (int c = 0; c < NC; ++c) asm volatile("" : "+v"(held[c]));
  };
  if (NC > 0) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (c * T + t < row.nvec) held[c] = row.template load<false>(c * T + t);
  }
  const float xone = one >= 0 ? elem<DT>(z, one) : -INFINITY;
  const float z0 = id0 >= 0 ? elem<DT>(z, id0) : 0.f;
  auto leave_named = [&] {
    if (t < 64) {
      nid[t] = id0;
      np[t] = p0;
      nz[t] = z0;
    }
  };
  if (NC > 0) leave_named();
  if (BWD) {
    st = Stat{a.stats[3 * r], a.stats[3 * r + 1], a.stats[3 * r + 2]};
  } else if (NC > 0) {
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
    st.m = scalar(block_max<T>(mx, red[0]));
    keep_packed();
    const float x1[1] = {xone};
    add<MODE>(st, x1, lt);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (c * T + t < row.nvec) {
        float x[N];
        W::unpack(held[c], x);
        add<MODE>(st, x, lt);
      }
    }
    if (has_hard(MODE)) st.s = block_sum<T>(st.s, red[1]);
    if (MODE == SOFT) st.t = block_sum<T>(st.t, red[1]);
    else if (MODE == BOTH_T1) st.t = st.s;
    else if (has_soft(MODE)) st.t = block_sum<T>(st.t, (float*)wred);
  } else {
    const float x1[1] = {xone};
    st.m = xone;
    add<MODE>(st, x1, lt);
    int k = t;
    for (; k + (U - 1) * T < row.nvec; k += U * T) {
      u32x4 raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = row.template load<NT>(k + u * T);
      float x[U][N], mx = st.m;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        W::unpack(raw[u], x[u]);
#pragma unroll
        for (int e = 0; e < N; ++e) mx = fmaxf(mx, x[u][e]);
      }
      rescale<MODE>(st, mx, lt);
#pragma unroll
      for (int u = 0; u < U; ++u) add<MODE>(st, x[u], lt);
    }
    for (; k < row.nvec; k += T) {
      float x[N], mx = st.m;
      W::unpack(row.template load<NT>(k), x);
#pragma unroll
      for (int e = 0; e < N; ++e) mx = fmaxf(mx, x[e]);
      rescale<MODE>(st, mx, lt);
      add<MODE>(st, x, lt);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
      st = join<MODE>(st, Stat{__shfl_xor(st.m, o, 64), __shfl_xor(st.s, o, 64), __shfl_xor(st.t, o, 64)}, lt);
    if ((t & 63) == 0) wred[t >> 6] = st;
    __syncthreads();
    st = wred[0];
    for (int i = 1; i < T / 64; ++i) st = join<MODE>(st, wred[i], lt);
  }
  if (!BWD) {  // the same in every thread: scalar registers
    st.m = scalar(st.m);
    st.s = scalar(st.s);
    st.t = scalar(st.t);
  }
  // without a pair the soft part is 0, which an infinite sum makes of its gradient
  if (!BWD && has_soft(MODE) && a.tsum[2 * r] == 0.f) st.t = INFINITY;
  if (PHASE == LOSS_FWD && t == 0) {
    a.stats[3 * r] = st.m;
    a.stats[3 * r + 1] = st.s;
    a.stats[3 * r + 2] = st.t;
  }
  // the row's loss, by the first wave
  auto row_loss = [&] {
    float cross = 0.f, zy = nz[0];  // sum p (m - z) / T; the label's logit, of thread 0
    if (has_soft(MODE)) {
      if (np[t] != 0.f) cross = np[t] * (st.m - nz[t]);
      for (int k = t + 64; k <= a.K; k += 64)
        if (prob[k] != 0.f) cross += prob[k] * (st.m - elem<DT>(z, place[k]));
      cross = wave_sum(cross) / a.T;
      if (has_hard(MODE) && t == 0 && !bad) zy = elem<DT>(z, y);
    }
    if (t == 0) {
      float loss = 0.f;
      if (has_soft(MODE) && st.t != INFINITY) loss = a.sw * a.T * a.T * (a.tsum[2 * r + 1] + cross + logf(st.t));
      if (has_hard(MODE) && !bad) loss += a.hw * ((st.m - zy) + logf(st.s));
      a.row_loss[r] = bad ? NAN : loss;
    }
  };
  if (NC == 0) leave_named();
  if (FWD) {
    if (t < 64) row_loss();
    return;
  }

  float c = a.factor;
  if (a.dloss) c *= a.dloss[a.reduction == PE_LOSS_NONE ? r : 0];
  if (a.count) c /= *a.count;
  if (bad) c = NAN;
  float ch = 0.f, ct = 0.f;
  if (has_hard(MODE)) ch = c * a.hw / st.s;
  if (has_soft(MODE)) ct = c * a.sw * a.T / st.t;
  c = scalar(c);
  ch = scalar(ch);
  ct = scalar(ct);
  auto dense = [&](float x) {
    float e, et;
    exps<MODE>(x - st.m, lt, e, et);
    if (MODE == HARD) return ch * e;
    if (MODE == SOFT) return ct * et;
    if (MODE == BOTH_T1) return (ch + ct) * e;
    if (MODE == BOTH_T2) return et * (ch * et + ct);
    return ch * e + ct * et;
  };
  auto piece = [&](int k, const u32x4& raw) {
    float x[N];
    W::unpack(raw, x);
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = dense(x[e]);
    store_piece<DT>(dbody, k, a.stream, x);
  };
  if (one >= 0) put<DT>(dz, one, dense(xone));
  if (NC > 0) {
    keep_packed();
#pragma unroll
    for (int k = 0; k < NC; ++k)
      if (k * T + t < row.nvec) piece(k * T + t, held[k]);
  } else {
    int k = t;
    for (; k + (U - 1) * T < row.nvec; k += U * T) {
      u32x4 raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = row.template load<false>(k + u * T);
#pragma unroll
      for (int u = 0; u < U; ++u) piece(k + u * T, raw[u]);
    }
    for (; k < row.nvec; k += T) piece(k, row.template load<false>(k));
  }
  __syncthreads();
  if (t >= 64) return;
  // the named places again
  auto named = [&](int32_t id, float x, float p) {
    if (id < 0) return;
    float g = dense(x);
    if (has_soft(MODE)) g -= c * a.sw * a.T * p;
    if (has_hard(MODE) && id == y) g -= c * a.hw;
    put<DT>(dz, id, g);
  };
  named(nid[t], nz[t], np[t]);
  if (has_soft(MODE))
    for (int k = t + 64; k <= a.K; k += 64)
      if (place[k] >= 0) named(place[k], elem<DT>(z, place[k]), prob[k]);
  if (!BWD) row_loss();
}

// The sum of the row losses in fp64 and the number of rows that count, by one workgroup of T threads, U rows a thread in
// flight.  The rows that count are the labels other than ignore_index, but with `shift` the first of every sequence,
// which is no row's.  L: the labels' type, or void for a sum alone.
template <bool SUM, int T, class L> __device__ __forceinline__ void add_rows(const LossArgs& a, double& s, int32_t& n) {
  constexpr bool COUNT = !std::is_void<L>::value;
  using Y = typename std::conditional<COUNT, L, int32_t>::type;
  const Y* lab = (const Y*)a.labels;
  const uint32_t rows = (uint32_t)a.rows, shift = (uint32_t)a.shift;
  constexpr int U = 8;
  for (uint32_t r0 = threadIdx.x; r0 < rows; r0 += U * T) {
    float x[U];
    Y y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t r = min(r0 + u * T, rows - 1);
      x[u] = SUM ? a.row_loss[r] : 0.f;
      y[u] = COUNT ? lab[r] : 0;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t r = r0 + u * T;
      s += r < rows ? x[u] : 0.f;
      n += COUNT && r < rows && (int64_t)y[u] != a.ignore && !(shift && r % shift == 0) ? 1 : 0;
    }
  }
}
template <bool SUM, bool COUNT, int T> __device__ __forceinline__ void reduce_rows(const LossArgs& a, float* loss, float* count) {
  __shared__ double rs[T / 64];
  __shared__ int32_t rn[T / 64];
  double s = 0.;
  int32_t n = 0;
  if (COUNT && a.labels && a.label_bytes == 8) add_rows<SUM, T, int64_t>(a, s, n);
  else if (COUNT && a.labels) add_rows<SUM, T, int32_t>(a, s, n);
  else if (SUM) add_rows<SUM, T, void>(a, s, n);
  if (!a.labels && threadIdx.x == 0) n = (int32_t)a.rows;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    if (SUM) s += __shfl_xor(s, o, 64);
    if (COUNT) n += __shfl_xor(n, o, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    rs[threadIdx.x >> 6] = s;
    rn[threadIdx.x >> 6] = n;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < T / 64; ++i) {
    s += rs[i];
    n += rn[i];
  }
  if (COUNT) *count = (float)n;
  if (SUM) *loss = (float)(a.reduction == PE_LOSS_MEAN ? s / (COUNT ? (double)n : (double)*count) : s);
}

__global__ __launch_bounds__(1024) void loss_count_kernel(LossArgs a, float* count) {
  reduce_rows<false, true, 1024>(a, nullptr, count);
}
// the count is formed here (COUNT) or was ahead of the rows
template <bool COUNT> __global__ __launch_bounds__(1024) void loss_reduce_kernel(LossArgs a, float* loss, float* count) {
  reduce_rows<true, COUNT, 1024>(a, loss, count);
}

// The teacher's pairs, ahead of the rows' workgroups, which would wait for them: a wave takes a row.  What the rows need
// of them (LossArgs::place, prob, tsum) is the places whose gradient is more than the dense one, that is every
// different id among the pairs present with the sum of its probabilities and behind them the label if it is none of
// them (-1 where there is none); whether any pair is present, P; and E = sum p ln p.
constexpr int TEACHER_ROWS = 4;
constexpr int teacher_pitch(int K) { return (K + 3) / 4 * 4; }

// what the wave's lanes wrote to LDS is there for the others
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ void teacher_row(const LossArgs& a, int64_t r, int32_t* tid, float* tp) {
  const int lane = threadIdx.x & 63, K = a.K, pitch = teacher_pitch(K);
  int64_t y;  // on its way beside the pairs; a row that does not count is not waited for
  const bool counts = row_label(a, (uint32_t)r, y);
  const float lt = LOG2E / a.T;
  float mx = -INFINITY;
  for (int k = lane; k < pitch; k += 64) {
    int64_t id = -1;
    float x = 0.f;
    if (k < K) {
      id = load_id(a.tid, a.tid_bytes, r * a.tid_rs + k);
      x = load_as_float(a.tlog, r * a.tlog_rs + k, a.tlog_dtype);
    }
    const bool have = id >= 0 && id < a.V && x != -INFINITY;
    tid[k] = have ? (int32_t)id : -1;
    tp[k] = x;
    if (have) mx = fmaxf(mx, x);
  }
  mx = wave_max(mx);
  float n = 0.f;
  for (int k = lane; k < K; k += 64)
    if (tid[k] >= 0) n += ex2((tp[k] - mx) * lt);
  n = wave_sum(n);
  const float ln = logf(n);
  float E = 0.f;
  for (int k = lane; k < K; k += 64) {
    float p = 0.f;
    if (tid[k] >= 0) {
      const float d = tp[k] - mx;
      p = ex2(d * lt) / n;
      if (p != 0.f) E += p * (d / a.T - ln);
    }
    tp[k] = p;
  }
  wave_sync();
  E = wave_sum(E);
  if (!counts || !a.labels || a.hw == 0.f || y < 0 || y >= a.V) y = -1;
  bool label = false;  // among the pairs
  int32_t* place = a.place + r * (K + 1);
  float* prob = a.prob + r * (K + 1);
  for (int k = lane; k < (K + 63) / 64 * 64; k += 64) {
    const int32_t id = k < K ? tid[k] : -1;
    bool first = id >= 0;
    int same = 0;
    for (int i = 0; i < pitch; i += 4) {
      const int4 o = *(const int4*)(tid + i);
      const bool s0 = o.x == id, s1 = o.y == id, s2 = o.z == id, s3 = o.w == id;
      same += (int)s0 + (int)s1 + (int)s2 + (int)s3;
      first = first && !((s0 && i < k) || (s1 && i + 1 < k) || (s2 && i + 2 < k) || (s3 && i + 3 < k));
    }
    float p = k < K ? tp[k] : 0.f;
    if (first && same > 1) {  // an id that comes twice
      p = 0.f;
      for (int i = 0; i < K; ++i) p += tid[i] == id ? tp[i] : 0.f;
    }
    if (k < K) {
      place[k] = first ? id : -1;
      prob[k] = first ? p : 0.f;
    }
    label = label || (id >= 0 && id == y);
  }
  label = __ballot(label) != 0;
  if (lane == 0) {
    place[K] = label ? -1 : (int32_t)y;
    prob[K] = 0.f;
    a.tsum[2 * r] = n != 0.f ? 1.f : 0.f;
    a.tsum[2 * r + 1] = E;
  }
}

// the teacher's rows; with `count` also the number of rows that count, by a workgroup ahead of them
__global__ __launch_bounds__(TEACHER_ROWS * 64) void loss_teacher_kernel(LossArgs a, float* count) {
  extern __shared__ __attribute__((aligned(16))) char dyn[];
  int64_t block = blockIdx.x;
  if (count && block-- == 0) {
    reduce_rows<false, true, TEACHER_ROWS * 64>(a, nullptr, count);
    return;
  }
  const int w = threadIdx.x >> 6, pitch = teacher_pitch(a.K);
  const int64_t r = block * TEACHER_ROWS + w;
  if (r < a.rows) teacher_row(a, r, (int32_t*)dyn + 2 * w * pitch, (float*)dyn + (2 * w + 1) * pitch);
}

template <int DT, int PHASE, int T, int NC, int U, int WPE = 1> static int run_loss(const LossArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)a.rows), block(T);
  if (a.rows * T > 0xffffffffll) return -2;  // a grid's threads are counted in 32 bits
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, block, 0, s, a); };
  if (a.sw == 0.f) go(loss_row_kernel<DT, PHASE, HARD, T, NC, U, WPE>);
  else if (a.hw == 0.f) go(loss_row_kernel<DT, PHASE, SOFT, T, NC, U, WPE>);
  else if (a.T == 1.f) go(loss_row_kernel<DT, PHASE, BOTH_T1, T, NC, U, WPE>);
  else if (a.T == 2.f) go(loss_row_kernel<DT, PHASE, BOTH_T2, T, NC, U, WPE>);
  else go(loss_row_kernel<DT, PHASE, BOTH, T, NC, U, WPE>);
  return hipGetLastError() == hipSuccess ? 0 : -7;
}

// Threads a row by its pieces.  The step holds the row in as few registers a thread as the threads allow, with as few
// rows in flight as keep the memory busy: the bf16 step of 8192 x 32000 takes 201 us with four workgroups of 512
// threads on a compute unit, 189 us with two of 1024; that of 4096 x 50257 189 us with one workgroup of 1024 threads
// and 100 registers, 164 us with two in 64 registers (waves a SIMD as the last argument; with a teacher these spill,
// 216 us, and two of 512 threads take 183); 4096 x 65536 230 us and, by two of 512 threads, 206 us; 2048 x 130000 244
// us held and 257 us read twice.  Forward and backward are within 4 % of these for 256 to 1024 threads and two to six
// pieces in flight, but for the backward, which 512 threads take 3 % longer.
template <int DT, int PHASE> static int run_loss(const LossArgs& a, hipStream_t s) {
  const int pieces = a.V / Vec<DT>::N;
  if constexpr (PHASE == LOSS_STEP) {
    if (pieces <= 64 * 4) return run_loss<DT, PHASE, 64, 4, 1>(a, s);
    if (pieces <= 256 * 4) return run_loss<DT, PHASE, 256, 4, 1>(a, s);
    if (pieces <= 512 * 4) return run_loss<DT, PHASE, 512, 4, 1>(a, s);
    if (pieces <= 1024 * 4) return run_loss<DT, PHASE, 1024, 4, 1, 8>(a, s);
    if (pieces <= 1024 * 7 && a.sw == 0.f) return run_loss<DT, PHASE, 1024, 7, 1, 8>(a, s);
    if (pieces <= 512 * 16) return run_loss<DT, PHASE, 512, 16, 1, 4>(a, s);
    if (pieces <= 1024 * 16) return run_loss<DT, PHASE, 1024, 16, 1, 4>(a, s);
    return run_loss<DT, PHASE, 1024, 0, 4>(a, s);
  } else {
    if (pieces <= 64 * 4) return run_loss<DT, PHASE, 64, 0, 4>(a, s);
    if (pieces <= 256 * 8) return run_loss<DT, PHASE, 256, 0, 4>(a, s);
    if constexpr (PHASE == LOSS_BWD) return run_loss<DT, PHASE, 1024, 0, 3>(a, s);
    else return run_loss<DT, PHASE, 512, 0, 4>(a, s);
  }
}

template <int DT> static int loss_phase(int phase, const LossArgs& a, hipStream_t s) {
  if (phase == LOSS_BWD) return run_loss<DT, LOSS_BWD>(a, s);
  if (phase == LOSS_STEP) return run_loss<DT, LOSS_STEP>(a, s);
  return a.stats ? run_loss<DT, LOSS_FWD>(a, s) : run_loss<DT, LOSS_ALONE>(a, s);
}

int launch_loss(int dtype, int phase, LossArgs a, hipStream_t s) {
  if (a.rows == 0) return 0;
  a.stream = a.rows * a.V * (dtype == 1 ? 4 : 2) > STREAM_BYTES;
  if (dtype == 0) return loss_phase<0>(phase, a, s);
  if (dtype == 1) return loss_phase<1>(phase, a, s);
  return loss_phase<2>(phase, a, s);
}

bool loss_has_teacher(const LossArgs& a) { return a.sw != 0.f; }

int launch_loss_prepare(const LossArgs& a, float* count, hipStream_t s) {
  if (a.rows > 0 && loss_has_teacher(a)) {
    const unsigned blocks = (unsigned)((a.rows + TEACHER_ROWS - 1) / TEACHER_ROWS) + (count ? 1 : 0);
    if ((int64_t)blocks * TEACHER_ROWS * 64 > 0xffffffffll) return -2;  // a grid's threads are counted in 32 bits
    hipLaunchKernelGGL(loss_teacher_kernel, dim3(blocks), dim3(TEACHER_ROWS * 64), 8 * TEACHER_ROWS * teacher_pitch(a.K), s, a,
                       count);
  } else if (count) {
    hipLaunchKernelGGL(loss_count_kernel, dim3(1), dim3(1024), 0, s, a, count);
  }
  return hipGetLastError() == hipSuccess ? 0 : -7;
}

int launch_loss_reduce(const LossArgs& a, float* loss, float* count, bool form_count, hipStream_t s) {
  if (form_count) hipLaunchKernelGGL(loss_reduce_kernel<true>, dim3(1), dim3(1024), 0, s, a, loss, count);
  else hipLaunchKernelGGL(loss_reduce_kernel<false>, dim3(1), dim3(1024), 0, s, a, loss, count);
  return hipGetLastError() == hipSuccess ? 0 : -7;
}

}  // namespace pe
