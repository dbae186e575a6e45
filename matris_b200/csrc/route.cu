// Router of a mixture of experts: softmax over a row's experts, its top_k, per-expert counts, balance loss, the grouping of the rows
// by expert, and the gradient; and the weighted sum that brings the experts' outputs back to their rows.
//
// A row is held by L neighbouring lanes, V experts each (L V >= n_experts), so that a warp works on 32 / L rows at once and a row's
// reductions take log2 L shuffles.  The selection is a chain of comparisons, and instructions bound it: with four experts a lane, 64-bit
// keys and expf, 573,894 rows of 32 experts took 89 us of this launch alone, with eight, 32-bit keys and the hardware's power of two 61.
// Choices are made on the logits' order-preserving bits; a lane keeps the first of its equal ones, lanes compare columns.
//
// Grouping without atomics whose order could matter: a block takes a run of rows and counts its choices per expert (k_route), the
// counts are scanned expert by expert (k_route_scan), and every block then gives its pairs their slots in row order
// (k_route_place).  Few rows take all three steps in one block (k_route_small).  The loss's sums of probabilities go the same way,
// float32 inside a block's lanes, float64 across blocks.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "row_math.cuh"

namespace mb {

constexpr int RT_THREADS = 256, RT_WARPS = RT_THREADS / 32;
constexpr int RT_MAX_EXPERTS = 1024, RT_MAX_K = 32;

struct RtArgs {
  int64_t n_rows, ld, ld_d, block_rows;
  int32_t n_experts, top_k, renorm, n_blocks;
  const void* logits;
  const uint8_t* valid;
  int32_t* ids; float* weights;
  int32_t* counts; float* loss;
  int32_t *offsets, *row_of, *slot_of;
  const float *dweights, *dloss;
  void* dlogits;
  double* p_total;   // [n_experts]
  float* p_part;     // [n_experts, n_blocks]
  int32_t* c_part;   // [n_experts + 1, n_blocks]: choices by expert, rows routed; after the scan the exclusive sums over the blocks
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ void from_float(float x, float& y) { y = x; }
__device__ __forceinline__ void from_float(float x, __nv_bfloat16& y) { y = __float2bfloat16_rn(x); }
__device__ __forceinline__ void from_float(float x, __half& y) { y = __float2half_rn(x); }

constexpr float MINUS_INF = -INFINITY;

// V logits of a row from column c on, -inf behind the last expert
template <typename T, int V, bool VEC> __device__ __forceinline__ void load_logits(const T* row, int c, int n, float (&x)[V]) {
  if constexpr (VEC) {  // n is a multiple of 4 and the rows are aligned to four values
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      if (c + i < n) {
        struct alignas(4 * sizeof(T)) Four { T v[4]; };
        const Four f = *reinterpret_cast<const Four*>(row + c + i);
#pragma unroll
        for (int q = 0; q < 4; ++q) x[i + q] = to_float(f.v[q]);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) x[i + q] = MINUS_INF;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = c + i < n ? to_float(row[c + i]) : MINUS_INF;
  }
}
template <typename T, int V, bool VEC> __device__ __forceinline__ void store_logits(T* row, int c, int n, const float (&x)[V]) {
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < V; i += 4)
      if (c + i < n) {
        struct alignas(4 * sizeof(T)) Four { T v[4]; } f;
#pragma unroll
        for (int q = 0; q < 4; ++q) from_float(x[i + q], f.v[q]);
        *reinterpret_cast<Four*>(row + c + i) = f;
      }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c + i < n) from_float(x[i], row[c + i]);
  }
}

template <int L> __device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int L> __device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// The logit's order as an unsigned number: 0 for an expert that is not available, NaN above everything, -0 equal to 0
__device__ __forceinline__ uint32_t choice_key(float x) {
  uint32_t u = __float_as_uint(x + 0.f);
  u = (u & 0x80000000u) ? ~u : u | 0x80000000u;
  if (x != x) u = 0xFFC00000u;
  return x == MINUS_INF ? 0 : u;
}
__device__ __forceinline__ float key_value(uint32_t u) { return __uint_as_float((u & 0x80000000u) ? u & 0x7FFFFFFFu : ~u); }
// the larger key of a row's lanes, of equal ones the one of the lower column
template <int L> __device__ __forceinline__ void lanes_best(uint32_t& key, int& column) {
#pragma unroll
  for (int o = 1; o < L; o <<= 1) {
    const uint32_t k = __shfl_xor_sync(0xffffffffu, key, o);
    const int c = __shfl_xor_sync(0xffffffffu, column, o);
    if (k > key || (k == key && c < column)) { key = k; column = c; }
  }
}
// exp(x), x <= 0: the hardware's power of two of x log2 e, off by some |x| 2^-24 (expf, exact to a step, took a third of a row's instructions)
__device__ __forceinline__ float exp_below(float x) { return __expf(x); }

// Rows [from, to) of a block: choices and weights to memory, choices counted in hist[], rows routed returned per thread, column sums
// of the probabilities left in cols[0 .. n_experts)
template <typename T, int L, int V, int Q, bool VEC>
__device__ __forceinline__ void route_rows(const RtArgs& a, int64_t from, int64_t to, int32_t* hist, float (*cols)[L * V]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % L, c0 = sub * V, n = a.n_experts, k = a.top_k;
  const T* const logits = static_cast<const T*>(a.logits);
  for (int i = threadIdx.x; i <= n; i += RT_THREADS) hist[i] = 0;
  __syncthreads();
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  int routed_rows = 0;
  constexpr int STEP = RT_THREADS / L;
  // The next row is asked for before this one is worked on: a row's selection is a chain of shuffles that leaves the loads time enough.
  float ahead[V];
  auto ask = [&](int64_t t) {
    const bool use = t < to && (!a.valid || a.valid[t]);
    if (use) load_logits<T, V, VEC>(logits + t * a.ld, c0, n, ahead);
    else
#pragma unroll
      for (int i = 0; i < V; ++i) ahead[i] = MINUS_INF;
  };
  ask(from + warp * (32 / L) + lane / L);
  for (int64_t t0 = from + warp * (32 / L); t0 < to; t0 += STEP) {  // the same for all lanes of a warp: shuffles need them
    const int64_t t = t0 + lane / L;
    const bool in = t < to;
    float x[V];
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = ahead[i];
    ask(t + STEP);
    uint32_t key[V];
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = choice_key(x[i]);
    int id[Q];       // this lane's choices: every L-th, Q >= top_k / L
    float e_of[Q];
    float m = 0.f, total = 0.f, chosen = 0.f;
    bool routed = false;
    for (int j = 0; j < k; ++j) {
      uint32_t best = key[0];
      int column = c0;
#pragma unroll
      for (int i = 1; i < V; ++i)
        if (key[i] > best) { best = key[i]; column = c0 + i; }
      lanes_best<L>(best, column);
      if (j == 0) {
        routed = best != 0;
        m = routed ? key_value(best) : 0.f;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) { x[i] = x[i] == MINUS_INF ? 0.f : exp_below(x[i] - m); s += x[i]; }
        total = lanes_sum<L>(s);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) key[i] = c0 + i == column ? 0 : key[i];
      const float e = best ? exp_below(key_value(best) - m) : 0.f;
      chosen += e;
#pragma unroll
      for (int q = 0; q < Q; ++q)
        if (j == q * L + sub) { id[q] = best ? column : -1; e_of[q] = e; }
    }
    if (in) {
      const float scale = routed ? 1.f / (a.renorm ? chosen : total) : 0.f;
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int j = q * L + sub;
        if (j < k) {
          a.ids[t * k + j] = id[q];
          a.weights[t * k + j] = id[q] < 0 ? 0.f : e_of[q] * scale;
          if (id[q] >= 0) atomicAdd(&hist[id[q]], 1);
        }
      }
    }
    if (routed) {
      const float inv = 1.f / total;
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = fmaf(x[i], inv, acc[i]);
      if (sub == 0) ++routed_rows;
    }
  }
#pragma unroll
  for (int o = L; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
  if (lane < L)
#pragma unroll
    for (int i = 0; i < V; ++i) cols[warp][c0 + i] = acc[i];
  if (routed_rows) atomicAdd(&hist[n], routed_rows);
  __syncthreads();
}

template <typename T, int L, int V, int Q, bool VEC> __global__ void __launch_bounds__(RT_THREADS) k_route(const __grid_constant__ RtArgs a) {
  pdl_sync();
  __shared__ int32_t hist[RT_MAX_EXPERTS + 1];
  __shared__ float cols[RT_WARPS][L * V];
  const int64_t from = min((int64_t)blockIdx.x * a.block_rows, a.n_rows), to = min(from + a.block_rows, a.n_rows);
  route_rows<T, L, V, Q, VEC>(a, from, to, hist, cols);
  for (int e = threadIdx.x; e <= a.n_experts; e += RT_THREADS) {
    a.c_part[(int64_t)e * a.n_blocks + blockIdx.x] = hist[e];
    if (e < a.n_experts) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < RT_WARPS; ++w) s += cols[w][e];
      a.p_part[(int64_t)e * a.n_blocks + blockIdx.x] = s;
    }
  }
}

// warp per expert (the last one: rows routed): totals, and the blocks' counts become exclusive sums
__global__ void __launch_bounds__(RT_THREADS) k_route_scan(const __grid_constant__ RtArgs a) {
  pdl_sync();
  const int e = blockIdx.x * RT_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (e > a.n_experts) return;
  int32_t* const c = a.c_part + (int64_t)e * a.n_blocks;
  const float* const p = a.p_part + (int64_t)e * a.n_blocks;
  // a lane takes a run of blocks: its sum, a scan over the lanes, then its exclusive sums
  const int per = (a.n_blocks + 31) / 32, b0 = min(lane * per, a.n_blocks), b1 = min(b0 + per, a.n_blocks);
  int32_t mine = 0;
  double sum = 0.;
#pragma unroll 8
  for (int b = b0; b < b1; ++b) mine += c[b];
  if (e < a.n_experts)
#pragma unroll 8
    for (int b = b0; b < b1; ++b) sum += (double)p[b];
  int32_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int32_t u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  const int32_t before = __shfl_sync(0xffffffffu, upto, 31);
  int32_t at = upto - mine;
#pragma unroll 8
  for (int b = b0; b < b1; ++b) {
    const int32_t v = c[b];
    c[b] = at;
    at += v;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) {
    a.counts[e] = before;
    if (e < a.n_experts) a.p_total[e] = sum;
  }
}

// base[e] = first slot of expert e, base[n] = slots in use, from the counts: by warp 0
__device__ __forceinline__ void first_slots(const int32_t* counts, int n, int32_t* base) {
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < 32) {
    int32_t before = 0;
    for (int e0 = 0; e0 < n; e0 += 32) {
      const int32_t v = e0 + lane < n ? counts[e0 + lane] : 0;
      int32_t s = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int32_t u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += u;
      }
      if (e0 + lane < n) base[e0 + lane] = before + s - v;
      before += __shfl_sync(0xffffffffu, s, 31);
    }
    if (lane == 0) base[n] = before;
  }
}

// Slots of the pairs of rows [from, to): each warp takes a run of pairs, counts it, and hands out slots in order from first[e] + the
// counts of the warps before it
__device__ __forceinline__ void place_pairs(const RtArgs& a, int64_t from, int64_t to, const int32_t* first, int32_t (*of_warp)[RT_MAX_EXPERTS]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = a.n_experts, k = a.top_k;
  const int64_t q0 = from * k, q1 = to * k, per = ((q1 - q0 + RT_WARPS * 32 - 1) / (RT_WARPS * 32)) * 32;
  const int64_t w0 = min(q0 + warp * per, q1), w1 = min(w0 + per, q1);
  for (int e = lane; e < n; e += 32) of_warp[warp][e] = 0;
  __syncwarp();
  for (int64_t q = w0 + lane; q < w1; q += 32) {
    const int e = a.ids[q];
    if (e >= 0) atomicAdd(&of_warp[warp][e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < n; e += RT_THREADS) {
    int32_t at = first[e];
#pragma unroll
    for (int w = 0; w < RT_WARPS; ++w) {
      const int32_t c = of_warp[w][e];
      of_warp[w][e] = at;
      at += c;
    }
  }
  __syncthreads();
  for (int64_t q = w0 + lane; q - lane < w1; q += 32) {
    const int e = q < w1 ? a.ids[q] : -1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int before = __popc(same & ((1u << lane) - 1u));
    int32_t slot = -1;
    if (e >= 0) slot = of_warp[warp][e] + before;
    __syncwarp();
    if (e >= 0 && before == 0) of_warp[warp][e] += __popc(same);
    __syncwarp();
    if (q < w1) {
      a.slot_of[q] = slot;
      if (e >= 0) a.row_of[slot] = (int32_t)(q / k);
    }
  }
}

__device__ __forceinline__ float balance_loss(double dot, int n_experts, int top_k, int32_t rows) {
  return rows > 0 ? (float)(dot * (double)n_experts / ((double)top_k * (double)rows * (double)rows)) : 0.f;
}
__device__ __forceinline__ double warp_sum_double(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__global__ void __launch_bounds__(RT_THREADS) k_route_place(const __grid_constant__ RtArgs a) {
  pdl_sync();
  __shared__ int32_t base[RT_MAX_EXPERTS + 1], of_warp[RT_WARPS][RT_MAX_EXPERTS];
  const int n = a.n_experts;
  first_slots(a.counts, n, base);
  __syncthreads();
  const int64_t used = base[n], all = a.n_rows * a.top_k;
  if (blockIdx.x == 0) {
    for (int e = threadIdx.x; e <= n; e += RT_THREADS) a.offsets[e] = base[e];
    if (threadIdx.x < 32) {
      double dot = 0.;
      for (int e = threadIdx.x; e < n; e += 32) dot += (double)a.counts[e] * a.p_total[e];
      dot = warp_sum_double(dot);
      if (threadIdx.x == 0) *a.loss = balance_loss(dot, n, a.top_k, a.counts[n]);
    }
    __syncthreads();
  }
  for (int64_t i = used + (int64_t)blockIdx.x * RT_THREADS + threadIdx.x; i < all; i += (int64_t)gridDim.x * RT_THREADS) a.row_of[i] = -1;
  __syncthreads();
  for (int e = threadIdx.x; e < n; e += RT_THREADS) base[e] += a.c_part[(int64_t)e * a.n_blocks + blockIdx.x];
  __syncthreads();
  const int64_t from = min((int64_t)blockIdx.x * a.block_rows, a.n_rows);
  place_pairs(a, from, min(from + a.block_rows, a.n_rows), base, of_warp);
}

template <typename T, int L, int V, int Q, bool VEC> __global__ void __launch_bounds__(RT_THREADS) k_route_small(const __grid_constant__ RtArgs a) {
  pdl_sync();
  __shared__ int32_t hist[RT_MAX_EXPERTS + 1], base[RT_MAX_EXPERTS + 1];
  constexpr int COLS = RT_WARPS * L * V * 4, OF = RT_WARPS * RT_MAX_EXPERTS * 4;
  __shared__ __align__(16) uint8_t both[COLS > OF ? COLS : OF];
  float (*cols)[L * V] = reinterpret_cast<float (*)[L * V]>(both);
  route_rows<T, L, V, Q, VEC>(a, 0, a.n_rows, hist, cols);
  const int n = a.n_experts;
  for (int e = threadIdx.x; e <= n; e += RT_THREADS) a.counts[e] = hist[e];
  first_slots(hist, n, base);
  if (threadIdx.x >= 32 && threadIdx.x < 64) {
    const int lane = threadIdx.x - 32;
    double dot = 0.;
    for (int e = lane; e < n; e += 32) {
      double s = 0.;
      for (int w = 0; w < RT_WARPS; ++w) s += (double)cols[w][e];
      dot += (double)hist[e] * s;
    }
    dot = warp_sum_double(dot);
    if (lane == 0) *a.loss = balance_loss(dot, n, a.top_k, hist[n]);
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= n; e += RT_THREADS) a.offsets[e] = base[e];
  for (int64_t i = base[n] + (int64_t)threadIdx.x; i < a.n_rows * a.top_k; i += RT_THREADS) a.row_of[i] = -1;
  place_pairs(a, 0, a.n_rows, base, reinterpret_cast<int32_t (*)[RT_MAX_EXPERTS]>(both));
}

template <typename T, int L, int V, int Q, bool VEC> __global__ void __launch_bounds__(RT_THREADS) k_route_bwd(const __grid_constant__ RtArgs a) {
  pdl_sync();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % L, c0 = sub * V, n = a.n_experts, k = a.top_k;
  const T* const logits = static_cast<const T*>(a.logits);
  T* const dlogits = static_cast<T*>(a.dlogits);
  float share[V];  // d loss / d p of this lane's experts
  const int32_t rows = a.counts[n];
  const double unit = a.dloss && rows > 0 ? (double)*a.dloss * (double)n / ((double)k * (double)rows * (double)rows) : 0.;
#pragma unroll
  for (int i = 0; i < V; ++i) share[i] = c0 + i < n ? (float)(unit * (double)a.counts[c0 + i]) : 0.f;
  const int64_t step = (int64_t)gridDim.x * (RT_THREADS / L), first = ((int64_t)blockIdx.x * RT_WARPS + warp) * (32 / L);
  int next_id[Q];  // the next row's, asked for before this one is worked on
  float next_dw[Q], next_w[Q], next_x[V];
  auto ask = [&](int64_t t) {
    const bool in = t < a.n_rows;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int j = q * L + sub;
      const bool use = in && j < k;
      next_id[q] = use ? a.ids[t * k + j] : -1;
      next_dw[q] = use && a.dweights ? a.dweights[t * k + j] : 0.f;
      next_w[q] = use && a.renorm ? a.weights[t * k + j] : 0.f;
    }
    if (in) load_logits<T, V, VEC>(logits + t * a.ld, c0, n, next_x);
    else
#pragma unroll
      for (int i = 0; i < V; ++i) next_x[i] = MINUS_INF;
  };
  ask(first + lane / L);
  for (int64_t t0 = first; t0 < a.n_rows; t0 += step) {
    const int64_t t = t0 + lane / L;
    const bool in = t < a.n_rows;
    int id[Q];
    float dw[Q], w[Q], x[V];
    float dot = 0.f;
#pragma unroll
    for (int q = 0; q < Q; ++q) id[q] = next_id[q];
#pragma unroll
    for (int q = 0; q < Q; ++q) { dw[q] = next_dw[q]; w[q] = next_w[q]; }
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = next_x[i];
    ask(t + step);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      if (id[q] < 0) dw[q] = w[q] = 0.f;
      else dot = fmaf(w[q], dw[q], dot);
    }
    // what a row that is not routed holds goes no further: its gradient is zero
    const bool routed = __shfl_sync(0xffffffffu, id[0], lane - sub) >= 0;
    float m = x[0];
#pragma unroll
    for (int i = 1; i < V; ++i) m = fmaxf(m, x[i]);
    m = lanes_max<L>(m);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) { x[i] = x[i] == MINUS_INF ? 0.f : exp_below(x[i] - m); s += x[i]; }
    s = lanes_sum<L>(s);
    const float inv = routed ? 1.f / s : 0.f;
    if (a.renorm) dot = lanes_sum<L>(dot);
    float g[V], extra[V];
#pragma unroll
    for (int i = 0; i < V; ++i) { g[i] = share[i]; extra[i] = 0.f; }
#pragma unroll
    for (int q = 0; q < Q; ++q)
      for (int j = 0; j < L && q * L + j < k; ++j) {
        const int e = __shfl_sync(0xffffffffu, id[q], lane - sub + j) - c0;
        const float dwj = __shfl_sync(0xffffffffu, dw[q], lane - sub + j);
        const float wj = a.renorm ? __shfl_sync(0xffffffffu, w[q], lane - sub + j) : 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (e == i) {
            if (a.renorm) extra[i] = wj * (dwj - dot);
            else g[i] += dwj;
          }
      }
    float mean = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) { x[i] *= inv; mean = fmaf(x[i], g[i], mean); }
    mean = lanes_sum<L>(mean);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = routed ? fmaf(x[i], g[i] - mean, extra[i]) : 0.f;
    if (in) store_logits<T, V, VEC>(dlogits + t * a.ld_d, c0, n, x);
  }
}

// ------------------------------------------------------------------ the experts' outputs back to their rows
struct CbArgs {
  int64_t n_rows, n_slots, ld_y, ld_out, ld_dout, ld_dy;
  int32_t top_k, width, n_experts;
  const int32_t *slot_of, *offsets;
  const float *weights, *y, *dout;
  float *out, *dy, *dweights;
};

// Warp per row, all rows at once: a row's loads hang on its slots, and the many warps hide both latencies (286,947 rows of 128, two
// choices, 441 MB: 94 us; warps that take rows in turn and ask for the next row's slots ahead 96 - 105)
__global__ void __launch_bounds__(RT_THREADS) k_combine(const __grid_constant__ CbArgs a) {
  pdl_sync();
  const int64_t t = (int64_t)blockIdx.x * RT_WARPS + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (t >= a.n_rows) return;
  for (int c = 4 * lane; c < a.width; c += 128) {
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int j = 0; j < a.top_k; ++j) {
      const int64_t slot = a.slot_of[t * a.top_k + j];
      if (slot < 0 || slot >= a.n_slots) continue;
      const float w = a.weights ? a.weights[t * a.top_k + j] : 1.f;
      const float4 v = ld4(a.y + slot * a.ld_y + c);
      s = make_float4(fmaf(w, v.x, s.x), fmaf(w, v.y, s.y), fmaf(w, v.z, s.z), fmaf(w, v.w, s.w));
    }
    st4(a.out + t * a.ld_out + c, s);
  }
}

// Backward a warp takes rows in turn (a row is three times the forward pass's traffic): lane j holds choice j's slot and weight, asked
// for a row ahead; four choices' rows are in flight (the same rows, 735 MB: 146 us; a row a warp 172).
struct Choices {
  int slot;     // -1: none
  float w;
  __device__ __forceinline__ void ask(const CbArgs& a, int64_t t, int lane, int64_t first, int64_t used) {
    slot = -1;
    w = 1.f;
    if (t < a.n_rows && lane < a.top_k) {
      slot = a.slot_of[t * a.top_k + lane];
      if (a.weights) w = a.weights[t * a.top_k + lane];
      if (slot < first || slot >= used) slot = -1;
    }
  }
};

__global__ void __launch_bounds__(RT_THREADS) k_combine_bwd(const __grid_constant__ CbArgs a) {
  pdl_sync();
  const int lane = threadIdx.x & 31;
  const int64_t step = (int64_t)gridDim.x * RT_WARPS, t0 = (int64_t)blockIdx.x * RT_WARPS + (threadIdx.x >> 5);
  int64_t first = 0, used = a.n_slots;  // slots of the experts; the others are no choice's, whoever names them
  if (a.offsets) {
    first = min(max((int64_t)a.offsets[0], (int64_t)0), a.n_slots);
    used = min(max((int64_t)a.offsets[a.n_experts], first), a.n_slots);
    const int64_t skip = used - first;
    for (int64_t i = t0; i < a.n_slots - skip; i += step) {
      const int64_t s = i < first ? i : i + skip;
      for (int c = 4 * lane; c < a.width; c += 128) st4(a.dy + s * a.ld_dy + c, make_float4(0.f, 0.f, 0.f, 0.f));
    }
  }
  Choices next;
  next.ask(a, t0, lane, first, used);
  for (int64_t t = t0; t < a.n_rows; t += step) {
    const Choices now = next;
    next.ask(a, t + step, lane, first, used);
    float mine = 0.f;  // lane j: dweights[t, j]
    for (int j0 = 0; j0 < a.top_k; j0 += 4) {
      float dot[4] = {0.f, 0.f, 0.f, 0.f};
      for (int c0 = 0; c0 < a.width; c0 += 128) {
        const int c = c0 + 4 * lane;
        const bool in = c < a.width;
        const float4 g = in ? ld4(a.dout + t * a.ld_dout + c) : make_float4(0.f, 0.f, 0.f, 0.f);
        float4 v[4];
        int slot[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          slot[i] = j0 + i < a.top_k ? __shfl_sync(0xffffffffu, now.slot, j0 + i) : -1;
          v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (slot[i] >= 0 && in && a.dweights) v[i] = ld4(a.y + (int64_t)slot[i] * a.ld_y + c);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float w = __shfl_sync(0xffffffffu, now.w, (j0 + i) & 31);
          if (slot[i] >= 0 && in) {
            st4(a.dy + (int64_t)slot[i] * a.ld_dy + c, scl4(g, w));
            dot[i] += dot4(g, v[i]);
          }
        }
      }
      if (a.dweights) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (j0 + i >= a.top_k) break;
          const float s = warp_sum(dot[i]);
          if (lane == j0 + i) mine = s;
        }
      }
    }
    if (a.dweights && lane < a.top_k) a.dweights[t * a.top_k + lane] = mine;
  }
}

// ------------------------------------------------------------------ host side
static int route_blocks(int64_t n_rows, int n_sm) {
  const int64_t most = 4 * (int64_t)n_sm, want = (n_rows + 63) / 64;
  return (int)(want < most ? (want > 0 ? want : 1) : most);
}
// Few rows: one block does everything.  (One block / three launches: 512 rows of 8 experts 10.2 / 12.3 us, 1,024 14.3 / 12.3, 2,048 22 / 12.3;
// 64 rows of 64, top 6 11.8 / 16.4, 256 26.6 / 16.4; 16 rows of 256, top 8 12.3 / 22, 64 33 / 43.)
static bool route_small(int64_t n_rows, int n_experts) { return n_rows * n_experts <= 4096; }
static bool route_valid(const mb_route* d) {
  return d && d->n_rows >= 0 && d->n_experts >= 1 && d->n_experts <= RT_MAX_EXPERTS && d->top_k >= 1 && d->top_k <= RT_MAX_K &&
         d->top_k <= d->n_experts && d->dtype >= 0 && d->dtype <= 2 && d->n_rows <= INT32_MAX / d->top_k;
}
static RtArgs route_args(const mb_route* d) {
  RtArgs a = {};
  a.n_rows = d->n_rows; a.ld = d->ld_logits; a.ld_d = d->ld_dlogits;
  a.n_experts = d->n_experts; a.top_k = d->top_k; a.renorm = d->renorm;
  a.logits = d->logits; a.valid = d->valid; a.ids = d->ids; a.weights = d->weights; a.counts = d->counts; a.loss = d->loss;
  a.offsets = d->offsets; a.row_of = d->row_of; a.slot_of = d->slot_of; a.dweights = d->dweights; a.dloss = d->dloss; a.dlogits = d->dlogits;
  return a;
}
static bool route_vector(const mb_route* d, const void* rows, int64_t ld) {
  const uintptr_t bytes = d->dtype == MB_DTYPE_F32 ? 16 : 8;
  return d->n_experts % 4 == 0 && ld % 4 == 0 && reinterpret_cast<uintptr_t>(rows) % bytes == 0;
}
// f.run<T, L, V, Q, VEC>(): lanes of a row by the number of experts, choices of a lane by top_k
template <typename T, int L, int V, bool VEC, typename F> static void route_choices(int k, F& f) {
  constexpr int most = L >= 32 ? 1 : L == 16 ? 2 : L == 8 ? 4 : 8;  // top_k <= 32 and <= L V
  if (k <= L) f.template run<T, L, V, 1, VEC>();
  else f.template run<T, L, V, most, VEC>();
}
template <typename T, bool VEC, typename F> static void route_lanes(int n, int k, F& f) {
  if (n <= 8) route_choices<T, 1, 8, VEC>(k, f);
  else if (n <= 16) route_choices<T, 2, 8, VEC>(k, f);
  else if (n <= 32) route_choices<T, 4, 8, VEC>(k, f);
  else if (n <= 64) route_choices<T, 8, 8, VEC>(k, f);
  else if (n <= 128) route_choices<T, 16, 8, VEC>(k, f);
  else if (n <= 256) route_choices<T, 32, 8, VEC>(k, f);
  else route_choices<T, 32, 32, VEC>(k, f);
}
template <typename F> static void route_typed(int dtype, bool vec, int n, int k, F f) {
  if (dtype == MB_DTYPE_F32) { if (vec) route_lanes<float, true>(n, k, f); else route_lanes<float, false>(n, k, f); }
  else if (dtype == MB_DTYPE_BF16) { if (vec) route_lanes<__nv_bfloat16, true>(n, k, f); else route_lanes<__nv_bfloat16, false>(n, k, f); }
  else { if (vec) route_lanes<__half, true>(n, k, f); else route_lanes<__half, false>(n, k, f); }
}
struct RouteFwd {
  const RtArgs& a; cudaStream_t st; bool small;
  template <typename T, int L, int V, int Q, bool VEC> void run() const {
    if (small) launch(k_route_small<T, L, V, Q, VEC>, 1, RT_THREADS, 0, st, a);
    else launch(k_route<T, L, V, Q, VEC>, (unsigned)a.n_blocks, RT_THREADS, 0, st, a);
  }
};
struct RouteBwd {
  const RtArgs& a; cudaStream_t st; int n_sm;
  template <typename T, int L, int V, int Q, bool VEC> void run() const {
    const int64_t want = (a.n_rows + RT_THREADS / L - 1) / (RT_THREADS / L), most = 8 * (int64_t)n_sm;
    launch(k_route_bwd<T, L, V, Q, VEC>, (unsigned)(want < most ? want : most), RT_THREADS, 0, st, a);
  }
};

}  // namespace mb

using namespace mb;

extern "C" size_t mb_route_scratch(int64_t n_rows, int32_t n_experts) {
  int n_sm = 0;
  if (n_rows < 0 || n_experts < 1 || route_small(n_rows, n_experts) || sm_count(&n_sm) != MB_OK) return 0;
  const size_t nb = (size_t)route_blocks(n_rows, n_sm);
  return 8 * (size_t)n_experts + 4 * nb * (2 * (size_t)n_experts + 1);
}

extern "C" int mb_route_fwd(const mb_route* d, void* stream) {
  if (!route_valid(d) || !d->counts || !d->loss || !d->offsets) return MB_ERR_INVALID;
  if (d->n_rows > 0 && (!d->logits || d->ld_logits < d->n_experts || !d->ids || !d->weights || !d->row_of || !d->slot_of))
    return MB_ERR_INVALID;
  const bool small = route_small(d->n_rows, d->n_experts);
  if (!small && (!d->scratch || (reinterpret_cast<uintptr_t>(d->scratch) & 15u))) return MB_ERR_INVALID;
  const cudaStream_t st = (cudaStream_t)stream;
  int n_sm = 0, rc = sm_count(&n_sm);
  if (rc) return rc;
  RtArgs a = route_args(d);
  a.n_blocks = route_blocks(d->n_rows, n_sm);
  a.block_rows = (d->n_rows + a.n_blocks - 1) / a.n_blocks;
  a.p_total = static_cast<double*>(d->scratch);
  a.p_part = reinterpret_cast<float*>(a.p_total + d->n_experts);
  a.c_part = reinterpret_cast<int32_t*>(a.p_part + (size_t)d->n_experts * a.n_blocks);
  route_typed(d->dtype, route_vector(d, d->logits, d->ld_logits), d->n_experts, d->top_k, RouteFwd{a, st, small});
  if (!small) {
    launch(k_route_scan, (unsigned)cdiv(d->n_experts + 1, RT_WARPS), RT_THREADS, 0, st, a);
    launch(k_route_place, (unsigned)a.n_blocks, RT_THREADS, 0, st, a);
  }
  MB_LAUNCH_CHECK("k_route");
  return MB_OK;
}

extern "C" int mb_route_bwd(const mb_route* d, void* stream) {
  if (!route_valid(d)) return MB_ERR_INVALID;
  if (d->n_rows == 0) return MB_OK;
  if (!d->logits || d->ld_logits < d->n_experts || !d->ids || !d->weights || !d->counts || !d->dlogits || d->ld_dlogits < d->n_experts)
    return MB_ERR_INVALID;
  int n_sm = 0, rc = sm_count(&n_sm);
  if (rc) return rc;
  const RtArgs a = route_args(d);
  const bool vec = route_vector(d, d->logits, d->ld_logits) && route_vector(d, d->dlogits, d->ld_dlogits);
  route_typed(d->dtype, vec, d->n_experts, d->top_k, RouteBwd{a, (cudaStream_t)stream, n_sm});
  MB_LAUNCH_CHECK("k_route_bwd");
  return MB_OK;
}

static bool rows16(const void* p, int64_t ld, int width) {
  return p && (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 4 == 0 && ld >= width;
}
static bool combine_valid(const mb_combine* d) {
  return d && d->n_rows >= 0 && d->n_slots >= 0 && d->n_slots <= INT32_MAX && d->top_k >= 1 && d->top_k <= RT_MAX_K && d->width >= 4 && d->width % 4 == 0 &&
         d->n_rows <= INT32_MAX / d->top_k && d->n_experts >= 0 && (d->n_rows == 0 || d->slot_of);
}
static CbArgs combine_args(const mb_combine* d) {
  CbArgs a = {};
  a.n_rows = d->n_rows; a.n_slots = d->n_slots; a.ld_y = d->ld_y; a.ld_out = d->ld_out; a.ld_dout = d->ld_dout; a.ld_dy = d->ld_dy;
  a.top_k = d->top_k; a.width = d->width; a.n_experts = d->n_experts; a.slot_of = d->slot_of; a.offsets = d->offsets;
  a.weights = d->weights; a.y = d->y; a.dout = d->dout; a.out = d->out; a.dy = d->dy; a.dweights = d->dweights;
  return a;
}

extern "C" int mb_experts_combine_fwd(const mb_combine* d, void* stream) {
  if (!combine_valid(d)) return MB_ERR_INVALID;
  if (d->n_rows == 0) return MB_OK;
  if (!rows16(d->out, d->ld_out, d->width) || (d->n_slots > 0 && !rows16(d->y, d->ld_y, d->width))) return MB_ERR_INVALID;
  launch(k_combine, (unsigned)cdiv(d->n_rows, RT_WARPS), RT_THREADS, 0, (cudaStream_t)stream, combine_args(d));
  MB_LAUNCH_CHECK("k_combine");
  return MB_OK;
}

extern "C" int mb_experts_combine_bwd(const mb_combine* d, void* stream) {
  if (!combine_valid(d)) return MB_ERR_INVALID;
  if (d->n_slots > 0 && (!rows16(d->dy, d->ld_dy, d->width) || (d->dweights && !rows16(d->y, d->ld_y, d->width)))) return MB_ERR_INVALID;
  if (d->n_rows > 0 && !rows16(d->dout, d->ld_dout, d->width)) return MB_ERR_INVALID;
  const int64_t warps = d->n_rows > 0 ? d->n_rows : (d->offsets ? d->n_slots : 0);
  if (warps == 0) return MB_OK;
  int n_sm = 0, rc = sm_count(&n_sm);
  if (rc) return rc;
  const int64_t want = (warps + RT_WARPS - 1) / RT_WARPS, most = 8 * (int64_t)n_sm;
  launch(k_combine_bwd, (unsigned)(want < most ? want : most), RT_THREADS, 0, (cudaStream_t)stream, combine_args(d));
  MB_LAUNCH_CHECK("k_combine_bwd");
  return MB_OK;
}
