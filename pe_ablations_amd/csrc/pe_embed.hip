// The scaled token embedding and its gradient (include/pe_vocab.h).
//
//     out[t] = weight[ids[t]] * scale        dweight[v] = scale * sum_{t: ids[t] = v} dy[t]
//
// Both are bound by memory.  The gradient sorts the tokens by id (stable, so each id's tokens stay in order), notes
// each id's run of tokens and sums whole chunks of sorted tokens that share one id ahead of time, and then adds up
// the run of every row of the vocabulary: each row of the gradient is written once, by one workgroup, rows without a
// token as zeros, and no sum depends on the order in which workgroups run.  Measured: the lookup of 16384 rows of 2048 in
// bf16 19 us (4.8 TB/s), the gradient of 65536 tokens, a quarter of them padding, in 32000 of them 98 us (rows 61, chunks
// 15, sort 22), of 4096 tokens in 50257 fp32 rows of 512 31 us (3.6 TB/s).
//
// A row of H elements is cut into pieces, a piece a lane: 16 bytes where the row length, the strides and the addresses
// are multiples of 16; else 16 bytes at any address, the last piece moved back to end with the row (its elements that
// the piece before has as well are worked out twice, to the same values); single elements in rows below 16 bytes.
// `lpr` lanes (a power of two) work on a row together, 256 / lpr rows at once in a workgroup, and rows longer than lpr
// pieces are cut into column slices.
#include <algorithm>
#include <type_traits>

#include "pe_common.h"
#include "pe_internal.h"

namespace pe {

namespace {

enum { ELEMENT = 0, ALIGNED = 1, ANYWHERE = 2 };

// a piece of a row of dtype DT as floats
template <int DT, int KIND> struct Piece {
  static constexpr int ES = DT == 1 ? 4 : 2, N = KIND == ELEMENT ? 1 : 16 / ES;
  using R = typename std::conditional<KIND != ELEMENT, u32x4,
                                      typename std::conditional<DT == 1, uint32_t, uint16_t>::type>::type;
  using M = typename std::conditional<KIND == ANYWHERE, u32x4_any, R>::type;  // as it lies in memory
  // the first element of piece c
  static __device__ __forceinline__ int first(const EmbedArgs& a, int c) { return KIND == ANYWHERE ? min(c * N, a.H - N) : c * N; }
  static __device__ __forceinline__ R load(const void* p, int64_t byte) { return *(const M*)((const char*)p + byte); }
  static __device__ __forceinline__ void unpack(const R& r, float (&x)[N]) {
    if constexpr (KIND == ELEMENT) {
      if constexpr (DT == 1) x[0] = __builtin_bit_cast(float, r);
      else x[0] = DT == 0 ? bf2f(r) : h2f(r);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = r[i];
        if constexpr (DT == 1) x[i] = __builtin_bit_cast(float, w);
        else if constexpr (DT == 0) {
          x[2 * i] = __builtin_bit_cast(float, w << 16);
          x[2 * i + 1] = __builtin_bit_cast(float, w & 0xffff0000u);
        } else {
          unpack_h2(w, x[2 * i], x[2 * i + 1]);
        }
      }
    }
  }
  static __device__ __forceinline__ void store(void* p, int64_t byte, const float (&x)[N], bool stream) {
    R r;
    if constexpr (KIND == ELEMENT) {
      if constexpr (DT == 1) r = __builtin_bit_cast(uint32_t, x[0]);
      else r = DT == 0 ? f2bf(x[0]) : f2h(x[0]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (DT == 1) r[i] = __builtin_bit_cast(uint32_t, x[i]);
        else if constexpr (DT == 0) r[i] = pack_bf2(x[2 * i], x[2 * i + 1]);
        else r[i] = pack_h2(x[2 * i], x[2 * i + 1]);
      }
    }
    M* q = (M*)((char*)p + byte);
    if (stream) {
      asm volatile("");  // on either side: else the compiler makes one plain store of the two
      __builtin_nontemporal_store((M)r, q);
      asm volatile("");
    } else {
      *q = r;
    }
  }
};

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

// ------------------------------------------------------------------ lookup
constexpr int LOOKUP_ROWS = 4;  // rows a group of lanes has in flight

template <int DT, int KIND> __global__ __launch_bounds__(256) void embed_fwd_kernel(EmbedArgs a) {
  using P = Piece<DT, KIND>;
  const int sub = threadIdx.x & (a.lpr - 1), grp = threadIdx.x / a.lpr, ng = 256 / a.lpr;
  const int64_t t0 = ((int64_t)blockIdx.x * ng + grp) * LOOKUP_ROWS;
  int64_t id[LOOKUP_ROWS];
#pragma unroll
  for (int i = 0; i < LOOKUP_ROWS; ++i) id[i] = t0 + i < a.n ? load_id(a.ids, a.id_bytes, t0 + i) : -1;
  for (int c = sub; c < a.pieces; c += a.lpr) {
    const int j = P::first(a, c);
    typename P::R r[LOOKUP_ROWS] = {};
#pragma unroll
    for (int i = 0; i < LOOKUP_ROWS; ++i)
      if (id[i] >= 0 && id[i] < a.V) r[i] = P::load(a.x, (id[i] * a.x_rs + j) * P::ES);
#pragma unroll
    for (int i = 0; i < LOOKUP_ROWS; ++i) {
      if (t0 + i >= a.n) break;
      float x[P::N];
      P::unpack(r[i], x);
#pragma unroll
      for (int e = 0; e < P::N; ++e) x[e] = id[i] >= 0 && id[i] < a.V ? product(x[e], a.scale) : NAN;
      P::store(a.y, ((t0 + i) * a.y_rs + j) * P::ES, x, a.stream);
    }
  }
}

// ------------------------------------------------------------------ sorting the tokens
// The key of a token: its id, or V (behind every row of the vocabulary) when its gradient goes nowhere.
__device__ __forceinline__ int32_t id_key(const EmbedArgs& a, int64_t id) {
  return id < 0 || id >= a.V || id == a.pad ? (int32_t)a.V : (int32_t)id;
}
__device__ __forceinline__ int32_t token_key(const EmbedArgs& a, int64_t t) { return id_key(a, load_id(a.ids, a.id_bytes, t)); }
// Keys of tokens t0, t0 + step, ... , -1 from a.n (> 0) on; both halves of every id are loaded ahead of any use.
template <int M> __device__ __forceinline__ void token_keys(const EmbedArgs& a, int t0, int step, int32_t (&key)[M]) {
  const int32_t* ids = (const int32_t*)a.ids;
  const int w = a.id_bytes / 4, n = (int)a.n;
  int32_t lo[M], hi[M];
#pragma unroll
  for (int i = 0; i < M; ++i) {
    const int64_t at = (int64_t)min(t0 + i * step, n - 1) * w;
    lo[i] = ids[at];
    hi[i] = ids[at + w - 1];
  }
#pragma unroll
  for (int i = 0; i < M; ++i) {
    const int64_t id = w == 2 ? (int64_t)((uint64_t)(uint32_t)hi[i] << 32 | (uint32_t)lo[i]) : (int64_t)lo[i];
    key[i] = t0 + i * step < n ? id_key(a, id) : -1;
  }
}

// no token of any id yet: thread i of `n`
__device__ __forceinline__ void clear_runs(const EmbedArgs& a, int64_t i, int64_t n) {
  for (; i < a.V; i += n) a.run[i] = int2{0, 0};
}

// Least significant digits first, `bits` of them a pass, tiles of 1024 tokens.  A pass counts each tile's digits, turns
// the counts into each tile's place within its digit, and moves the tokens.  Up to FEW_TILES tiles add up the counts
// of those before them where they move the tokens; a launch of its own does so for more.
constexpr int TILE = 1024, MAXBITS = 10, FEW_TILES = 64;

struct SortArgs {
  const int32_t *key_in, *order_in;  // NULL in the first pass, which takes the tokens themselves
  int32_t *key_out, *order_out;
  int32_t *hist;                     // [tiles][bins], past FEW_TILES tiles then each one's offset within the bin
  int32_t *total;                    // [bins]
  int tiles, shift, bits;
};

__device__ __forceinline__ int32_t sort_key(const EmbedArgs& a, const SortArgs& s, int64_t i) {
  return s.key_in ? s.key_in[i] : token_key(a, i);
}

__global__ __launch_bounds__(TILE) void embed_hist_kernel(EmbedArgs a, SortArgs s) {
  __shared__ int32_t h[1 << MAXBITS];
  const int bins = 1 << s.bits, t = threadIdx.x;
  const int64_t i = (int64_t)blockIdx.x * TILE + t;
  if (!s.key_in) clear_runs(a, i, (int64_t)gridDim.x * TILE);
  if (t < bins) h[t] = 0;
  __syncthreads();
  if (i < a.n) atomicAdd(&h[(sort_key(a, s, i) >> s.shift) & (bins - 1)], 1);
  __syncthreads();
  if (t < bins) s.hist[(int64_t)blockIdx.x * bins + t] = h[t];
}

// a workgroup takes 32 bins; its 32 rows of threads each take a run of tiles
__global__ __launch_bounds__(1024) void embed_scan_kernel(SortArgs s) {
  __shared__ int32_t part[32][33];
  const int bins = 1 << s.bits, c = threadIdx.x & 31, j = threadIdx.x >> 5, b = blockIdx.x * 32 + c;
  const int per = (s.tiles + 31) / 32, k0 = min(j * per, s.tiles), k1 = min(k0 + per, s.tiles);
  int32_t sum = 0;
  if (b < bins)
    for (int k = k0; k < k1; ++k) sum += s.hist[(int64_t)k * bins + b];
  part[j][c] = sum;
  __syncthreads();
  int32_t run = 0;
  for (int i = 0; i < j; ++i) run += part[i][c];
  if (b >= bins) return;
  if (j == 31) s.total[b] = run + sum;
  for (int k = k0; k < k1; ++k) {
    const int32_t x = s.hist[(int64_t)k * bins + b];
    s.hist[(int64_t)k * bins + b] = run;
    run += x;
  }
}

// The stable place of a token in its tile: in a wave, the lanes below with the same digit (found by one ballot per bit);
// between waves, a count per wave and digit in LDS.
__global__ __launch_bounds__(TILE) void embed_scatter_kernel(EmbedArgs a, SortArgs s) {
  __shared__ uint16_t cnt[TILE / 64][1 << MAXBITS];
  __shared__ int32_t base[1 << MAXBITS], wsum[TILE / 64];
  const int bins = 1 << s.bits, t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int64_t i = (int64_t)blockIdx.x * TILE + t;
  // where each digit begins: an exclusive sum of the totals over the bins, one bin a thread
  int32_t tot = 0, ahead = 0;
  if (t < bins) {
    if (s.tiles <= FEW_TILES) {
#pragma unroll 16
      for (int k = 0; k < s.tiles; ++k) {
        const int32_t x = s.hist[k * bins + t];
        tot += x;
        ahead += k < (int)blockIdx.x ? x : 0;
      }
    } else {
      tot = s.total[t];
      ahead = s.hist[(int64_t)blockIdx.x * bins + t];
    }
  }
  int32_t inc = tot;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int32_t x = __shfl_up(inc, o, 64);
    if (lane >= o) inc += x;
  }
  if (lane == 63) wsum[w] = inc;
  for (int k = t; k < (TILE / 64) * (1 << MAXBITS) / 2; k += TILE) ((uint32_t*)cnt)[k] = 0;
  __syncthreads();
  int32_t before = 0;
  for (int k = 0; k < w; ++k) before += wsum[k];
  if (t < bins) base[t] = before + inc - tot + ahead;
  const bool live = i < a.n;
  const int32_t key = live ? sort_key(a, s, i) : 0;
  const int d = (key >> s.shift) & (bins - 1);
  uint64_t same = __ballot(live);
  for (int bit = 0; bit < s.bits; ++bit) {
    const uint64_t m = __ballot((d >> bit) & 1);
    same &= (d >> bit) & 1 ? m : ~m;
  }
  const int below = __popcll(same & ((1ull << lane) - 1));
  if (live && below == 0) cnt[w][d] = (uint16_t)__popcll(same);
  __syncthreads();
  if (t < bins) {
    uint32_t run = 0;
#pragma unroll
    for (int k = 0; k < TILE / 64; ++k) {
      const uint32_t x = cnt[k][t];
      cnt[k][t] = (uint16_t)run;
      run += x;
    }
  }
  __syncthreads();
  if (live) {
    const int32_t place = base[d] + cnt[w][d] + below;
    s.key_out[place] = key;
    s.order_out[place] = s.order_in ? s.order_in[i] : (int32_t)i;
  }
}

// ------------------------------------------------------------------ sums of rows
// Rows first, first + 1, ... of a list, added in order with `U` loads in flight
template <int DT, int KIND, int U = 8, class F>
__device__ __forceinline__ void add_rows(const void* x, int64_t col, int64_t first, int64_t end, F row, float (&s)[Piece<DT, KIND>::N]) {
  using P = Piece<DT, KIND>;
  int64_t i = first;
  for (; i + U <= end; i += U) {
    typename P::R r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) r[u] = P::load(x, row(i + u) + col);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[P::N];
      P::unpack(r[u], v);
#pragma unroll
      for (int e = 0; e < P::N; ++e) s[e] += v[e];
    }
  }
  for (; i < end; ++i) {
    float v[P::N];
    P::unpack(P::load(x, row(i) + col), v);
#pragma unroll
    for (int e = 0; e < P::N; ++e) s[e] += v[e];
  }
}

// the sums of chunks k, k + 1, ... behind one another, four of them in flight
template <int N> __device__ __forceinline__ void add_sums(const EmbedArgs& a, int j, int32_t k, int32_t end, float (&s)[N]) {
  const float* p = a.part + j;
  for (; k + 4 <= end; k += 4) {
    float x[4][N];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) x[u][e] = p[(int64_t)(k + u) * a.H + e];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) s[e] += x[u][e];
  }
  for (; k < end; ++k)
#pragma unroll
    for (int e = 0; e < N; ++e) s[e] += p[(int64_t)k * a.H + e];
}

// A chunk of a.chunk sorted tokens: notes where runs begin and end in it, and if all of it has one id adds up its
// rows, the workgroup's groups of lanes taking a run of tokens each and their sums added in order.
template <int DT, int KIND> __global__ __launch_bounds__(256) void embed_chunk_kernel(EmbedArgs a) {
  using P = Piece<DT, KIND>;
  const int slice = blockIdx.x % a.slices, bx = blockIdx.x / a.slices;  // a row's slices side by side
  const int64_t c0 = (int64_t)bx * a.chunk, c1 = c0 + a.chunk;
  if (slice == 0) {
    for (int64_t i = c0 + threadIdx.x; i < min(c1, a.n); i += 256) {
      const int32_t key = a.key[i], prev = i ? a.key[i - 1] : -1, next = i + 1 < a.n ? a.key[i + 1] : -1;
      if (key == (int32_t)a.V) break;
      if (key != prev) a.run[key].x = (int32_t)i;
      if (key != next) a.run[key].y = (int32_t)i + 1;
    }
  }
  if (c1 > a.n) return;
  const int32_t key = a.key[c0];
  if (key == (int32_t)a.V || a.key[c1 - 1] != key) return;
  const int sub = threadIdx.x & (a.lpr - 1), grp = threadIdx.x / a.lpr, ng = 256 / a.lpr;
  const int c = slice * a.lpr + sub;
  __shared__ float red[256 * P::N];
  float s[P::N] = {};
  const int64_t i0 = c0 + (int64_t)a.chunk * grp / ng, i1 = c0 + (int64_t)a.chunk * (grp + 1) / ng;
  if (c < a.pieces)
    add_rows<DT, KIND, 16>(a.x, (int64_t)P::first(a, c) * P::ES, i0, i1, [&](int64_t i) { return (int64_t)a.order[i] * a.x_rs * P::ES; }, s);
#pragma unroll
  for (int e = 0; e < P::N; ++e) red[threadIdx.x * P::N + e] = s[e];
  __syncthreads();
  if (grp == 0 && c < a.pieces) {
    for (int g = 1; g < ng; ++g)
#pragma unroll
      for (int e = 0; e < P::N; ++e) s[e] += red[(g * a.lpr + sub) * P::N + e];
#pragma unroll
    for (int e = 0; e < P::N; ++e) a.part[(int64_t)bx * a.H + P::first(a, c) + e] = s[e];
  }
}

constexpr int SHORT_RUN = 32;  // tokens that one group of lanes adds up alone
constexpr int MAX_ROWS = 64;   // rows of the vocabulary a workgroup takes

// The gradient's rows v = bx + j G, j < nr, of one workgroup from their runs of tokens: frequent ids are neighbours, and
// so are shared out.  Each group of lanes takes the rows with short runs in turn; then the workgroup adds up each long
// run together, as the tokens ahead of its first whole chunk, the chunks' sums (CHUNKS), and the tokens behind the
// last, cut into as many equal parts as there are groups, whose sums are added in order.
template <int DT, int KIND, bool CHUNKS, class O>
__device__ __forceinline__ void grad_rows(const EmbedArgs& a, int slice, int bx, int64_t G, int nr, const int2* run, float* red, O order) {
  using P = Piece<DT, KIND>;
  const int sub = threadIdx.x & (a.lpr - 1), grp = threadIdx.x / a.lpr, ng = 256 / a.lpr;
  const int c = slice * a.lpr + sub;
  const int j0 = P::first(a, c);
  const int64_t col = (int64_t)j0 * P::ES;
  auto token = [&](int64_t i) { return (int64_t)order(i) * a.x_rs * P::ES; };
  auto put = [&](int j, float (&s)[P::N]) {
#pragma unroll
    for (int e = 0; e < P::N; ++e) s[e] = product(s[e], a.scale);
    P::store(a.y, (bx + j * G) * a.y_rs * P::ES + col, s, a.stream);
  };
  if (c < a.pieces) {
    for (int j = grp; j < nr; j += ng) {
      const int32_t i0 = run[j].x, i1 = run[j].y;
      if (i1 - i0 > SHORT_RUN) continue;
      float s[P::N] = {};
      add_rows<DT, KIND, 4>(a.x, col, i0, i1, token, s);
      put(j, s);
    }
  }
  for (int j = 0; j < nr; ++j) {
    const int32_t i0 = run[j].x, i1 = run[j].y;
    if (i1 - i0 <= SHORT_RUN) continue;
    // items: [0, h) tokens i0.., [h, h + m) chunks k0.., [h + m, total) tokens behind the last chunk
    const int32_t k0 = CHUNKS ? (i0 + a.chunk - 1) / a.chunk : 0, k1 = CHUNKS ? i1 / a.chunk : 0;
    const bool chunks = k1 > k0;
    const int32_t h = chunks ? k0 * a.chunk - i0 : i1 - i0, m = chunks ? k1 - k0 : 0;
    const int32_t total = chunks ? h + m + (i1 - k1 * a.chunk) : h;
    const int32_t b0 = (int32_t)((int64_t)total * grp / ng), b1 = (int32_t)((int64_t)total * (grp + 1) / ng);
    float s[P::N] = {};
    if (c < a.pieces) {
      add_rows<DT, KIND>(a.x, col, i0 + min(b0, h), i0 + min(b1, h), token, s);
      if (chunks) {
        add_sums<P::N>(a, j0, k0 + min(max(b0 - h, 0), m), k0 + min(max(b1 - h, 0), m), s);
        const int64_t q = (int64_t)k1 * a.chunk - h - m;  // item b behind the chunks is token q + b
        add_rows<DT, KIND>(a.x, col, q + max(b0, h + m), q + max(b1, h + m), token, s);
      }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < P::N; ++e) red[threadIdx.x * P::N + e] = s[e];
    __syncthreads();
    if (grp == 0 && c < a.pieces) {
      for (int g = 1; g < ng; ++g)
#pragma unroll
        for (int e = 0; e < P::N; ++e) s[e] += red[(g * a.lpr + sub) * P::N + e];
      put(j, s);
    }
  }
}

// Bound by the latency of the tokens' rows, so by how many waves a SIMD holds and how many workgroups there are (bf16
// 32000 x 2048, 16384 / 65536 tokens, the whole gradient: 69 / 124 us with eight rows in flight in 87 registers and
// 1024 workgroups, 58 / 115 us with four in 64, 58 / 112 us with 2048 workgroups, 65 / 114 us with 4096).
template <int DT, int KIND>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(8))) void embed_bwd_kernel(EmbedArgs a) {
  const int slice = blockIdx.x % a.slices, bx = blockIdx.x / a.slices;
  __shared__ int2 run[MAX_ROWS];
  __shared__ float red[256 * Piece<DT, KIND>::N];
  const int64_t G = gridDim.x / a.slices;
  const int nr = (int)((a.V - bx + G - 1) / G);
  if (threadIdx.x < nr) run[threadIdx.x] = a.run[bx + threadIdx.x * G];
  __syncthreads();
  grad_rows<DT, KIND, true>(a, slice, bx, G, nr, run, red, [&](int64_t i) { return a.order[i]; });
}

// Up to FEW tokens, in one launch without a workspace: every workgroup picks the tokens of its own rows from all of them
// (G a power of two: row j of token id has id = bx + j G), in order, by a ballot for 64 tokens, and then lists each
// row's in turn.
constexpr int FEW = 4096;

template <int DT, int KIND> __global__ __launch_bounds__(256) void embed_bwd_few_kernel(EmbedArgs a, int log_g) {
  constexpr int N = Piece<DT, KIND>::N;
  const int slice = blockIdx.x % a.slices, bx = blockIdx.x / a.slices;
  __shared__ int2 run[MAX_ROWS];
  __shared__ uint16_t order[FEW];
  __shared__ union { uint32_t list[FEW]; float red[256 * N]; } u;  // j << 16 | token; the sums come after its last use
  __shared__ int32_t count[4];
  const int64_t G = (int64_t)1 << log_g;
  const int nr = (int)((a.V - bx + G - 1) / G), n = (int)a.n;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint64_t below = (1ull << lane) - 1;
  // wave w takes a quarter of the tokens, in whole steps of 64
  constexpr int STEPS = FEW / 256;
  const int steps = (n + 255) / 256, s0 = w * steps * 64;
  int32_t key[STEPS];
  if (n > 0) {
    token_keys(a, s0 + lane, 64, key);
  } else {
#pragma unroll
    for (int i = 0; i < STEPS; ++i) key[i] = -1;
  }
  int mine = 0;
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    if (i >= steps || key[i] >= (int32_t)a.V || (key[i] & (int32_t)(G - 1)) != bx) key[i] = -1;
    mine += __popcll(__ballot(key[i] >= 0));
  }
  if (lane == 0) count[w] = mine;
  __syncthreads();
  int at = 0;
  for (int i = 0; i < w; ++i) at += count[i];
  const int total = count[0] + count[1] + count[2] + count[3];
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const uint64_t m = __ballot(key[i] >= 0);
    if (key[i] >= 0) u.list[at + __popcll(m & below)] = (uint32_t)(key[i] >> log_g) << 16 | (uint32_t)(s0 + i * 64 + lane);
    at += __popcll(m);
  }
  __syncthreads();
  // the tokens of each row: wave w lists rows w, w + 4, ...; the rows before it say where it begins
  for (int j = w; j < nr; j += 4) {
    int before = 0, len = 0;
    for (int i = lane; i < (total + 63) / 64 * 64; i += 64) {
      const uint32_t x = i < total ? u.list[i] : 0xffffffffu;
      before += __popcll(__ballot((int)(x >> 16) < j));
      len += __popcll(__ballot((int)(x >> 16) == j));
    }
    if (len) {
      int pos = before;
      for (int i = lane; i < (total + 63) / 64 * 64; i += 64) {
        const uint32_t x = i < total ? u.list[i] : 0xffffffffu;
        const uint64_t m = __ballot((int)(x >> 16) == j);
        if ((int)(x >> 16) == j) order[pos + __popcll(m & below)] = (uint16_t)x;
        pos += __popcll(m);
      }
    }
    if (lane == 0) run[j] = int2{before, before + len};
  }
  __syncthreads();
  grad_rows<DT, KIND, false>(a, slice, bx, G, nr, run, u.red, [&](int64_t i) { return (int32_t)order[i]; });
}

namespace {

int piece_kind(int es, const EmbedArgs& a) {
  const uint64_t all = (uint64_t)(uintptr_t)a.x | (uintptr_t)a.y | (uint64_t)(a.x_rs * es) | (uint64_t)(a.y_rs * es) |
                       (uint64_t)((int64_t)a.H * es);
  return all % 16 == 0 ? ALIGNED : ((int64_t)a.H * es >= 16 ? ANYWHERE : ELEMENT);
}
int pieces_of(int kind, int H, int es) { return kind == ELEMENT ? H : (int)(((int64_t)H * es + 15) / 16); }

template <class F> int with_piece(int dtype, int kind, F&& f) {
  using std::integral_constant;
  auto go = [&](auto dt) {
    if (kind == ALIGNED) return f(dt, integral_constant<int, ALIGNED>{});
    if (kind == ANYWHERE) return f(dt, integral_constant<int, ANYWHERE>{});
    return f(dt, integral_constant<int, ELEMENT>{});
  };
  if (dtype == 0) return go(integral_constant<int, 0>{});
  if (dtype == 1) return go(integral_constant<int, 1>{});
  return go(integral_constant<int, 2>{});
}

// lanes a row: the power of two that covers its pieces, from 8 up to `most`
int lanes_per_row(int pieces, int most) {
  int l = 8;
  while (l < most && l < pieces) l *= 2;
  return l;
}

int64_t up4(int64_t n) { return (n + 3) / 4 * 4; }

// Sorted tokens a chunk: 64, and more where there would be over 512 chunks, whose sums one id may have to add up (65536
// tokens of one id, bf16 x 1024: 124 us with 64 and the sums one by one, 69 us with 128 and four in flight; of 32000
// ids, x 2048: 124 and 123 us).
int chunk_tokens(int64_t n) {
  int c = 64;
  while (c < 1024 && n / c > 512) c *= 2;
  return c;
}

int key_bits(int64_t V) {  // of keys 0 .. V
  int b = 1;
  while ((int64_t)1 << b <= V) ++b;
  return b;
}

// Outputs beyond this size are stored past the 256 MB cache, smaller ones left in it for their reader (the gradient of
// 32000 x 2048 in bf16, 125 MB, 16384 tokens: 58 and 48 us; of 50257 x 512 in fp32, 98 MB: 44 and 47 us).  The gradient of
// a few tokens, nearly all zeros, never is (the former with 2048 tokens: 32 us streamed, 29 us not).
bool streams(int64_t rows, int H, int es) { return rows * H * es > (112ll << 20); }

// a grid's threads are counted in 32 bits
bool grid_fits(int64_t blocks, int threads) { return blocks * threads <= 0xffffffffll; }

int done() { return hipGetLastError() == hipSuccess ? 0 : -7; }

}  // namespace

int launch_embed_fwd(int dtype, EmbedArgs a, hipStream_t s) {
  const int es = dtype == 1 ? 4 : 2, kind = piece_kind(es, a);
  a.pieces = pieces_of(kind, a.H, es);
  a.lpr = lanes_per_row(a.pieces, 256);
  a.stream = streams(a.n, a.H, es);
  const int64_t rows = (int64_t)(256 / a.lpr) * LOOKUP_ROWS;
  const dim3 grid((unsigned)((a.n + rows - 1) / rows)), block(256);
  if (!grid_fits((a.n + rows - 1) / rows, 256)) return -2;
  return with_piece(dtype, kind, [&](auto dt, auto v) {
    hipLaunchKernelGGL((embed_fwd_kernel<decltype(dt)::value, decltype(v)::value>), grid, block, 0, s, a);
    return done();
  });
}

// past FEW tokens: each id's run; [key][order] of the sorted tokens, twice; the digits' counts; the chunks' sums
int64_t embed_bwd_workspace(int64_t n, int64_t V, int H) {
  if (n <= FEW) return 0;
  return 4 * (up4(2 * V) + 4 * up4(n) + (((n + TILE - 1) / TILE + 1) << MAXBITS) + n / chunk_tokens(n) * (int64_t)H) + 16;
}

int launch_embed_bwd(int dtype, EmbedArgs a, void* ws, hipStream_t s) {
  const int es = dtype == 1 ? 4 : 2, kind = piece_kind(es, a);
  a.pieces = pieces_of(kind, a.H, es);
  // Lanes on a row: a whole workgroup where most rows of the gradient are zeros, so that the tokens are picked for
  // all of its columns at once; else a wave, whose slices and groups share the long runs (fp32 50257 x 512, 4096
  // tokens: 29 against 37 us; bf16 2000 x 1024, 4096 tokens: 24 against 18 us)
  a.lpr = lanes_per_row(a.pieces, a.n <= FEW && a.V >= 4 * a.n ? 256 : 64);
  a.slices = (a.pieces + a.lpr - 1) / a.lpr;
  a.stream = a.n > FEW && streams(a.V, a.H, es);
  if (a.n <= FEW) {
    // 15 to 30 rows a workgroup, fewer where that leaves compute units idle
    int log_g = 0;
    while (((int64_t)15 << (log_g + 1)) <= a.V || (log_g < 9 && ((int64_t)2 << log_g) <= a.V)) ++log_g;
    if (!grid_fits((int64_t)a.slices << log_g, 256)) return -2;
    return with_piece(dtype, kind, [&](auto dt, auto v) {
      hipLaunchKernelGGL((embed_bwd_few_kernel<decltype(dt)::value, decltype(v)::value>), dim3((unsigned)a.slices << log_g),
                         dim3(256), 0, s, a, log_g);
      return done();
    });
  }
  int32_t* p = (int32_t*)ws;
  auto take = [&](int64_t n) { int32_t* q = p; p += n; return q; };
  a.run = (int2*)take(up4(2 * a.V));
  a.key = take(up4(a.n));
  a.order = take(up4(a.n));
  int32_t *key2 = take(up4(a.n)), *order2 = take(up4(a.n));
  SortArgs o;
  o.tiles = (int)((a.n + TILE - 1) / TILE);
  o.hist = take((int64_t)o.tiles << MAXBITS);
  o.total = take(1 << MAXBITS);
  const int bits = key_bits(a.V), passes = (bits + MAXBITS - 1) / MAXBITS;
  o.bits = (bits + passes - 1) / passes;
  for (int i = 0; i < passes; ++i) {
    const bool last_in_first = (passes - 1 - i) % 2 == 0;  // the last pass writes a.key / a.order
    o.key_in = i == 0 ? nullptr : (last_in_first ? key2 : a.key);
    o.order_in = i == 0 ? nullptr : (last_in_first ? order2 : a.order);
    o.key_out = last_in_first ? a.key : key2;
    o.order_out = last_in_first ? a.order : order2;
    o.shift = i * o.bits;
    hipLaunchKernelGGL(embed_hist_kernel, dim3(o.tiles), dim3(TILE), 0, s, a, o);
    if (o.tiles > FEW_TILES)
      hipLaunchKernelGGL(embed_scan_kernel, dim3(((1 << o.bits) + 31) / 32), dim3(1024), 0, s, o);
    hipLaunchKernelGGL(embed_scatter_kernel, dim3(o.tiles), dim3(TILE), 0, s, a, o);
  }
  if (hipGetLastError() != hipSuccess) return -7;
  a.part = (float*)p;
  a.chunk = chunk_tokens(a.n);
  const unsigned chunks = (unsigned)((a.n + a.chunk - 1) / a.chunk);
  const unsigned rows = (unsigned)((a.V + MAX_ROWS - 1) / MAX_ROWS);
  const unsigned grid = (unsigned)std::min<int64_t>(a.V, std::max<int64_t>(rows, 2048));
  if (!grid_fits((int64_t)std::max(grid, chunks) * a.slices, 256)) return -2;
  return with_piece(dtype, kind, [&](auto dt, auto v) {
    constexpr int D = decltype(dt)::value, B = decltype(v)::value;
    hipLaunchKernelGGL((embed_chunk_kernel<D, B>), dim3(chunks * a.slices), dim3(256), 0, s, a);
    hipLaunchKernelGGL((embed_bwd_kernel<D, B>), dim3(grid * a.slices), dim3(256), 0, s, a);
    return done();
  });
}

}  // namespace pe
