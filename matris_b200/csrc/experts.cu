// Dense layers of a mixture of experts on rows grouped by expert: forward and data gradient (one product), weight gradient.
#include "row_math.cuh"

namespace mb {

constexpr int EX_MAX_EXPERTS = 1024, EX_MAX_WIDTH = 1024;

// Slots of an expert, whatever the offsets hold
__device__ __forceinline__ void expert_slots(const mb_experts& d, int e, int64_t& from, int64_t& to) {
  from = min(max((int64_t)d.offsets[e], (int64_t)0), d.n_slots);
  to = min(max((int64_t)d.offsets[e + 1], from), d.n_slots);
}
__device__ __forceinline__ const float* source_row(const mb_experts& d, int64_t s) {
  const int64_t r = d.idx ? min(max((int64_t)d.idx[s], (int64_t)0), d.n_rows - 1) : s;
  return d.x + r * d.ld_x;
}

// ------------------------------------------------------------------ float32 cores, the cross-check of the tensor-core ones
// 64 slots x 64 columns a block; row tiles are numbered through the experts, at most slots / 64 + experts of them
constexpr int ES_TILE = 64, ES_K = 16, ES_THREADS = 256;

__global__ void __launch_bounds__(ES_THREADS) k_experts_simt(const __grid_constant__ mb_experts d) {
  pdl_sync();
  __shared__ float xs[ES_K][ES_TILE + 4], ws[ES_K][ES_TILE + 4];
  int64_t from = 0, to = 0, tile = blockIdx.x;
  int e = 0;
  for (; e < d.n_experts; ++e) {
    expert_slots(d, e, from, to);
    const int64_t n = (to - from + ES_TILE - 1) / ES_TILE;
    if (tile < n) break;
    tile -= n;
  }
  const int c0 = blockIdx.y * ES_TILE, tid = threadIdx.x;
  if (e == d.n_experts) {
    if (d.zero_rest) {  // a block past the last tile clears its share of the rows behind the last slot
      const int64_t used = min(max((int64_t)d.offsets[d.n_experts], (int64_t)0), d.n_slots);
      for (int64_t s = used + tile * ES_TILE + tid / 16; s < min(used + (tile + 1) * ES_TILE, d.n_slots); s += ES_THREADS / 16)
        st4(d.y + s * d.ld_y + c0 + 4 * (tid % 16), make_float4(0.f, 0.f, 0.f, 0.f));
    }
    return;
  }
  const int64_t s0 = from + tile * ES_TILE;
  const int lr = tid / 4, lk = 4 * (tid % 4), ty = tid / 16, tx = tid % 16;
  const float* const xrow = source_row(d, min(s0 + lr, to - 1));
  const float* const wrow = d.w + ((int64_t)e * d.n_out + c0 + lr) * d.n_in;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < d.n_in; k0 += ES_K) {
    float4 v = ld4(xrow + k0 + lk);
    if (d.in_act) v = make_float4(silu_f(v.x), silu_f(v.y), silu_f(v.z), silu_f(v.w));
    const float4 w = ld4(wrow + k0 + lk);
    __syncthreads();
    xs[lk][lr] = v.x; xs[lk + 1][lr] = v.y; xs[lk + 2][lr] = v.z; xs[lk + 3][lr] = v.w;
    ws[lk][lr] = w.x; ws[lk + 1][lr] = w.y; ws[lk + 2][lr] = w.z; ws[lk + 3][lr] = w.w;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ES_K; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xs[k][4 * ty + i], ws[k][4 * tx + j], acc[i][j]);
  }
  const int c = c0 + 4 * tx;
  const float4 b = d.bias ? ld4(d.bias + (int64_t)e * d.n_out + c) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t s = s0 + 4 * ty + i;
    if (s >= to) break;
    float v[4] = {acc[i][0] + b.x, acc[i][1] + b.y, acc[i][2] + b.z, acc[i][3] + b.w};
    if (d.gate) {
      const float4 z = ld4(d.gate + s * d.ld_gate + c);
      v[0] *= silu_grad_f(z.x); v[1] *= silu_grad_f(z.y); v[2] *= silu_grad_f(z.z); v[3] *= silu_grad_f(z.w);
    }
    if (d.out_act)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = silu_f(v[j]);
    st4(d.y + s * d.ld_y + c, make_float4(v[0], v[1], v[2], v[3]));
  }
}

// 64 x 64 of one expert's gradient a block, its slots in order; the first column of blocks sums the bias gradient on the way
__global__ void __launch_bounds__(ES_THREADS) k_experts_grad_simt(const __grid_constant__ mb_experts d) {
  pdl_sync();
  __shared__ float gs[ES_K][ES_TILE + 4], xs[ES_K][ES_TILE + 4];
  const int e = blockIdx.z, n0 = blockIdx.y * ES_TILE, k0 = blockIdx.x * ES_TILE, tid = threadIdx.x;
  int64_t from, to;
  expert_slots(d, e, from, to);
  const int lr = tid / 16, lc = 4 * (tid % 16), ty = tid / 16, tx = tid % 16;
  float acc[4][4] = {}, db[4] = {};
  for (int64_t s0 = from; s0 < to; s0 += ES_K) {
    const int64_t s = s0 + lr;
    float4 g = make_float4(0.f, 0.f, 0.f, 0.f), v = g;
    if (s < to) {
      g = ld4(d.dy + s * d.ld_dy + n0 + lc);
      v = ld4(source_row(d, s) + k0 + lc);
      if (d.in_act) v = make_float4(silu_f(v.x), silu_f(v.y), silu_f(v.z), silu_f(v.w));
    }
    __syncthreads();
    st4(&gs[lr][lc], g);
    st4(&xs[lr][lc], v);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ES_K; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float gv = gs[k][4 * ty + i];
        db[i] += gv;
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(gv, xs[k][4 * tx + j], acc[i][j]);
      }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t n = (int64_t)e * d.n_out + n0 + 4 * ty + i;
    st4(d.dw + n * d.n_in + k0 + 4 * tx, make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]));
    if (d.dbias && blockIdx.x == 0 && tx == 0) d.dbias[n] = db[i];
  }
}

static bool aligned_rows(const void* p, int64_t ld, int width) {
  return p && (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 4 == 0 && ld >= width;
}
static bool experts_valid(const mb_experts* d) {
  return d && d->n_slots >= 0 && d->n_slots <= INT32_MAX && d->n_rows >= 0 && d->n_experts >= 1 && d->n_experts <= EX_MAX_EXPERTS &&
         d->n_in >= 128 && d->n_in <= EX_MAX_WIDTH && d->n_in % 128 == 0 && d->n_out >= 128 && d->n_out <= EX_MAX_WIDTH && d->n_out % 128 == 0 &&
         d->offsets && (d->n_slots == 0 || (aligned_rows(d->x, d->ld_x, d->n_in) && (d->idx ? d->n_rows >= 1 : d->n_rows >= d->n_slots)));
}

}  // namespace mb

using namespace mb;

extern "C" int mb_experts_linear(const mb_experts* d, void* stream) {
  if (!experts_valid(d) || !aligned_rows(d->w, d->n_in, d->n_in)) return MB_ERR_INVALID;
  if (d->bias && !aligned_rows(d->bias, d->n_out, d->n_out)) return MB_ERR_INVALID;
  if (d->n_slots == 0) return MB_OK;
  if (!aligned_rows(d->y, d->ld_y, d->n_out) || (d->gate && !aligned_rows(d->gate, d->ld_gate, d->n_out))) return MB_ERR_INVALID;
  const int64_t tiles = (d->n_slots + ES_TILE - 1) / ES_TILE + d->n_experts;
  launch(k_experts_simt, dim3((unsigned)tiles, (unsigned)(d->n_out / ES_TILE)), ES_THREADS, 0, (cudaStream_t)stream, *d);
  MB_LAUNCH_CHECK("k_experts_simt");
  return MB_OK;
}

extern "C" size_t mb_experts_grad_scratch(int64_t n_slots, int32_t n_experts, int32_t n_in, int32_t n_out) {
  (void)n_slots; (void)n_experts; (void)n_in; (void)n_out;
  return 0;
}

extern "C" int mb_experts_grad_w(const mb_experts* d, void* stream) {
  if (!experts_valid(d) || !aligned_rows(d->dw, d->n_in, d->n_in)) return MB_ERR_INVALID;
  if (d->n_slots > 0 && !aligned_rows(d->dy, d->ld_dy, d->n_out)) return MB_ERR_INVALID;
  const dim3 grid((unsigned)(d->n_in / ES_TILE), (unsigned)(d->n_out / ES_TILE), (unsigned)d->n_experts);
  launch(k_experts_grad_simt, grid, ES_THREADS, 0, (cudaStream_t)stream, *d);
  MB_LAUNCH_CHECK("k_experts_grad_simt");
  return MB_OK;
}
