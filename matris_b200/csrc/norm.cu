// Group norm over the rows of every structure, with an optional SiLU, forward and backward.
//
// A segment is a range of rows (a structure of a batch), a group a run of Cg = channels / groups neighbouring channels; statistics
// go over all values of a (segment, group), in float32 whatever the rows' type:
//   xh = (x - mean) rstd, z = xh w + b, y = z or SiLU(z)
//   dz = dy or dy SiLU'(z), g = dz w, dx = rstd (g - <g> - xh <g xh>), dw = sum dz xh, db = sum dz   (< >: mean over the (segment, group))
//
// Variances come from deviations, never from sums of squares: a thread takes eight rows of its channels at a time, their mean and
// their squared deviations from it, and joins such pairs by  M2 = M2a + M2b + (ma - mb)^2 na nb / (na + nb).  One pass over the
// data, and an offset of 1e4 standard deviations costs no more than the inputs' own rounding.
//
// Two ways through the data.  Segments of up to `limit` rows: one block takes a segment's slab (whole groups, 128 bytes of a row
// where that is possible), statistics first and then the rows again, which are in the caches by then.  Longer ones: blocks take
// chunks of rows, their partial statistics are joined in row order, and a third launch applies them.  Nothing is summed by atomics:
// the same call gives the same bits.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <string.h>
#include <initializer_list>
#include <type_traits>
#include "common.cuh"

namespace mb {

constexpr int GN_THREADS = 256, GN_WARPS = GN_THREADS / 32;
constexpr int GN_BATCH = 8;              // rows of a thread in flight, forward
template <int V> constexpr int gn_pairs = V == 8 ? 2 : 4;  // ... and backward, of two tensors: eight 16-bit values a piece cost registers
constexpr int GN_PLACES = 2;             // blocks of a multiprocessor that work by chunks
constexpr int GN_MAX_CHANNELS = 1024;  // 256 threads, four channels each

struct GnArgs {
  int64_t n_rows, ld_x, ld_y, ld_dy, ld_dx;
  const int32_t* seg_ptr;  // NULL: segments of n_rows / n_seg rows
  int32_t n_seg, channels, groups, act, zero_rest;
  int32_t slab_groups;     // groups of a block's slab
  int32_t limit;           // segments with more rows go by chunks; -1: all of them
  int32_t chunk;           // rows of a chunk
  float eps;
  const void *x, *dy;
  const float *w, *b;
  void *y, *dx;
  float* stats;            // [n_seg, groups, 2]: mean, rstd
  float* part;             // chunks' partial results: [chunks + n_seg, groups or channels, 2], chunk c and segment s in row c + s
  float* sums;             // backward: [n_seg, channels, 2]: sum dz, sum dz xh
};

// Blocks of a multiprocessor: three of the float32 forward pass, two of the others.  (573,894 float32 rows of 128 in 512 segments, eight
// groups, when this was chosen: forward 138 us with three, 150 with two or four; backward 256 with two, 274 with three.  Now 131 and 235.)
constexpr int gn_blocks(int v, bool forward = false) { return forward && v != 8 ? 3 : 2; }
template <typename T, int V> struct Vec;
template <> struct Vec<float, 4> { float4 r; };
template <> struct Vec<float, 1> { float r; };
template <typename T> struct Vec<T, 8> { uint4 r; };
template <> struct Vec<__nv_bfloat16, 1> { __nv_bfloat16 r; };
template <> struct Vec<__half, 1> { __half r; };

__device__ __forceinline__ void unpack(const Vec<float, 4>& v, float (&f)[4]) { f[0] = v.r.x; f[1] = v.r.y; f[2] = v.r.z; f[3] = v.r.w; }
__device__ __forceinline__ void unpack(const Vec<float, 1>& v, float (&f)[1]) { f[0] = v.r; }
__device__ __forceinline__ void unpack(const Vec<__nv_bfloat16, 1>& v, float (&f)[1]) { f[0] = __bfloat162float(v.r); }
__device__ __forceinline__ void unpack(const Vec<__half, 1>& v, float (&f)[1]) { f[0] = __half2float(v.r); }
__device__ __forceinline__ void unpack(const Vec<__nv_bfloat16, 8>& v, float (&f)[8]) {
  const uint32_t w[4] = {v.r.x, v.r.y, v.r.z, v.r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
}
__device__ __forceinline__ void unpack(const Vec<__half, 8>& v, float (&f)[8]) {
  const uint32_t w[4] = {v.r.x, v.r.y, v.r.z, v.r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = t.x; f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ void pack(const float (&f)[4], Vec<float, 4>& v) { v.r = make_float4(f[0], f[1], f[2], f[3]); }
__device__ __forceinline__ void pack(const float (&f)[1], Vec<float, 1>& v) { v.r = f[0]; }
__device__ __forceinline__ void pack(const float (&f)[1], Vec<__nv_bfloat16, 1>& v) { v.r = __float2bfloat16_rn(f[0]); }
__device__ __forceinline__ void pack(const float (&f)[1], Vec<__half, 1>& v) { v.r = __float2half_rn(f[0]); }
__device__ __forceinline__ void pack(const float (&f)[8], Vec<__nv_bfloat16, 8>& v) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&t);
  }
  v.r = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void pack(const float (&f)[8], Vec<__half, 8>& v) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 t = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&t);
  }
  v.r = make_uint4(w[0], w[1], w[2], w[3]);
}

// Rows of a segment, whatever the offsets hold: inside the tensor and never negative in number
__device__ __forceinline__ void segment_rows(const GnArgs& a, int64_t s, int64_t& from, int64_t& to) {
  if (a.seg_ptr) {
    from = min(max((int64_t)a.seg_ptr[s], (int64_t)0), a.n_rows);
    to = min(max((int64_t)a.seg_ptr[s + 1], from), a.n_rows);
  } else {
    const int64_t n = a.n_rows / a.n_seg;
    from = s * n;
    to = from + n;
  }
}
__device__ __forceinline__ bool by_chunks(const GnArgs& a, int64_t rows) { return rows > a.limit; }

// Arithmetic on a thread's V neighbouring channels, two float32 values at a time where there are two.  SiLU by the hardware's
// exponential and reciprocal (a few steps of float32): with expf and a division a value takes some 40 instructions, and 73 million of
// them 70 us of the 210 that this forward pass took.
template <int V> __device__ __forceinline__ void add_to(float (&a)[V], const float (&b)[V]) {
  if constexpr (V == 1) a[0] += b[0];
  else
#pragma unroll
    for (int c = 0; c < V; c += 2) apart(two(a[c], a[c + 1]) + two(b[c], b[c + 1]), a[c], a[c + 1]);
}
// a += (b - m)^2
template <int V> __device__ __forceinline__ void square_to(float (&a)[V], const float (&b)[V], const float (&m)[V]) {
  if constexpr (V == 1) { const float d = b[0] - m[0]; a[0] = fmaf(d, d, a[0]); }
  else
#pragma unroll
    for (int c = 0; c < V; c += 2) {
      const f2 d = less(two(b[c], b[c + 1]), two(m[c], m[c + 1]));
      apart(fma2(d, d, two(a[c], a[c + 1])), a[c], a[c + 1]);
    }
}

// Where a thread stands in a block that covers `width` channels from `c0` on: vector columns tx + 256 j, rows ty + TY i
template <int V> struct Place {
  int cols, tx_n, ty_n, tx, ty;
  bool used;
  __device__ __forceinline__ Place(int width) {
    cols = width / V;
    tx_n = min(cols, GN_THREADS);
    ty_n = GN_THREADS / tx_n;
    tx = threadIdx.x % tx_n;
    ty = threadIdx.x / tx_n;
    used = ty < ty_n;
  }
};

// Statistics of a block's rows and channels by thread: n rows, means and squared deviations of its channels
template <int W> struct Moments {
  float n, mean[W], m2[W];
  __device__ __forceinline__ void clear() {
    n = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) mean[i] = m2[i] = 0.f;
  }
};
__device__ __forceinline__ void join(float& na, float& ma, float& sa, float nb, float mb_, float sb) {
  const float n = na + nb, f = n > 0.f ? __fdividef(nb, n) : 0.f, d = mb_ - ma;
  ma = fmaf(d, f, ma);
  sa = sa + sb + d * d * na * f;
}

// A block's shared memory: per-channel pairs of every warp or row lane, and the groups' results
template <int W> struct GnShared {
  float first[GN_THREADS * W], second[GN_THREADS * W];  // [entries][width]
  float count[GN_THREADS];
  float group[2][GN_MAX_CHANNELS];
};

// A thread's rows of [from, to), n of them, `step` bytes apart.  f(q, rows, whole) for its batches of U rows: `whole` is true_type where all
// U are there, so that the bulk of the loop has no comparisons (with 64-bit row numbers compared and multiplied for every access a value
// took 34 instructions in the forward pass, and the multiprocessors issued every other cycle at half the copy rate).
template <int V> __device__ __forceinline__ int thread_rows(const Place<V>& p, int64_t from, int64_t to) {
  return p.used && to - from > p.ty ? (int)((to - from - p.ty + p.ty_n - 1) / p.ty_n) : 0;
}
template <int U, typename F> __device__ __forceinline__ void batches(int n, F f) {
  int left = n;
  for (; left >= U; left -= U) f(U, std::true_type{});
  if (left > 0) f(left, std::false_type{});
}
// The second pass reads and writes for the last time: both are marked so, which leaves L2 to the rows that the second pass is still to
// find there (573,894 rows of 512 bytes in 512 segments: that step took the forward pass from 148 to 138 us, the backward one from 301 to 274).
template <typename T, int V> struct Stream {
  const char* p;
  int64_t step;
  __device__ __forceinline__ Stream(const void* base, int64_t ld, const Place<V>& at, int64_t from, int c)
      : p(reinterpret_cast<const char*>(static_cast<const T*>(base) + (from + at.ty) * ld + c)), step((int64_t)sizeof(T) * ld * at.ty_n) {}
  template <int U, typename W> __device__ __forceinline__ void read(Vec<T, V> (&v)[U], int rows, W) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (W::value || i < rows) v[i] = *reinterpret_cast<const Vec<T, V>*>(p);
      p += step;
    }
  }
  __device__ __forceinline__ void write(const Vec<T, V>& v) {
    if constexpr (V > 1) {
      uint4 w;
      memcpy(&w, &v, 16);
      __stcs(reinterpret_cast<uint4*>(const_cast<char*>(p)), w);
    } else
      *reinterpret_cast<Vec<T, V>*>(const_cast<char*>(p)) = v;
    p += step;
  }
  template <int U, typename W> __device__ __forceinline__ void read_last(Vec<T, V> (&v)[U], int rows, W) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (W::value || i < rows) {
        if constexpr (V > 1) { const uint4 w = __ldcs(reinterpret_cast<const uint4*>(p)); memcpy(&v[i], &w, 16); }
        else v[i] = *reinterpret_cast<const Vec<T, V>*>(p);
      }
      p += step;
    }
  }
};

// means and squared deviations of [from, to) x [c0, c0 + width) into sh.group[0 / 1][group of the slab]
template <typename T, int V, int NC>
__device__ void block_stats(const GnArgs& a, GnShared<V * NC>& sh, int64_t from, int64_t to, int c0, int width, int cg) {
  const Place<V> p(width);
  const int rows = thread_rows(p, from, to);
  const float n_rows = (float)rows;
  Moments<V * NC> m;
  m.clear();
  if (rows > 0) {
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int cv = p.tx + GN_THREADS * j;
      if (NC > 1 && cv >= p.cols) break;
      Stream<T, V> x(a.x, a.ld_x, p, from, c0 + cv * V);
      float n = 0.f;
      batches<GN_BATCH>(rows, [&](int count, auto whole) {
        Vec<T, V> v[GN_BATCH];
        x.read(v, count, whole);
        const float nb = (float)count, inv = __fdividef(1.f, nb), f = __fdividef(nb, n + nb);
        float sum[V], dev[V];
#pragma unroll
        for (int c = 0; c < V; ++c) sum[c] = dev[c] = 0.f;
#pragma unroll
        for (int i = 0; i < GN_BATCH; ++i) {
          float t[V];
          unpack(v[i], t);
          if (decltype(whole)::value || i < count) add_to<V>(sum, t);
        }
#pragma unroll
        for (int c = 0; c < V; ++c) sum[c] *= inv;
#pragma unroll
        for (int i = 0; i < GN_BATCH; ++i) {
          float t[V];
          unpack(v[i], t);
          if (decltype(whole)::value || i < count) square_to<V>(dev, t, sum);
        }
#pragma unroll
        for (int c = 0; c < V; ++c) {
          const int k = V * j + c;
          const float d = sum[c] - m.mean[k];
          m.mean[k] = fmaf(d, f, m.mean[k]);
          m.m2[k] += dev[c] + d * d * n * f;
        }
        n += nb;
      });
    }
  }
  float n = n_rows;
  // lanes of a warp that hold the same channels, then warps (or row lanes) in shared memory
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool fold = p.tx_n < 32 && (p.tx_n & (p.tx_n - 1)) == 0;
  if (fold) {
    for (int o = p.tx_n; o < 32; o <<= 1) {
      const float nb = __shfl_xor_sync(0xffffffffu, n, o);
      const float na = n;
#pragma unroll
      for (int k = 0; k < V * NC; ++k) {
        float mb_ = __shfl_xor_sync(0xffffffffu, m.mean[k], o), sb = __shfl_xor_sync(0xffffffffu, m.m2[k], o);
        // both partners join in the same order, so that they hold the same bits
        const bool low_lane = (lane & o) == 0;
        float n1 = low_lane ? na : nb, m1 = low_lane ? m.mean[k] : mb_, s1 = low_lane ? m.m2[k] : sb;
        join(n1, m1, s1, low_lane ? nb : na, low_lane ? mb_ : m.mean[k], low_lane ? sb : m.m2[k]);
        m.mean[k] = m1; m.m2[k] = s1;
      }
      n = na + nb;
    }
  }
  const int entries = fold ? GN_WARPS : p.ty_n, e = fold ? warp : p.ty;
  __syncthreads();  // the previous use of the shared arrays is over
  if (p.used && (!fold || lane < p.tx_n)) {
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int cv = p.tx + GN_THREADS * j;
      if (NC > 1 && cv >= p.cols) break;
#pragma unroll
      for (int c = 0; c < V; ++c) {
        sh.first[e * width + cv * V + c] = m.mean[V * j + c];
        sh.second[e * width + cv * V + c] = m.m2[V * j + c];
      }
    }
    if (p.tx == 0) sh.count[e] = n;
  }
  __syncthreads();
  const float total = (float)(to - from) * (float)cg;
  for (int g = warp; g < width / cg; g += GN_WARPS) {
    float s = 0.f;
    for (int i = lane; i < entries * cg; i += 32) s = fmaf(sh.count[i / cg], sh.first[i / cg * width + g * cg + i % cg], s);
    const float mean = total > 0.f ? warp_sum(s) / total : 0.f;
    s = 0.f;
    for (int i = lane; i < entries * cg; i += 32) {
      const int at_ = i / cg * width + g * cg + i % cg;
      const float d = sh.first[at_] - mean;
      s += sh.second[at_] + d * d * sh.count[i / cg];
    }
    s = warp_sum(s);
    if (lane == 0) { sh.group[0][g] = mean; sh.group[1][g] = s; }
  }
  __syncthreads();
}

// A thread's channels: the numbers that a row needs.  (Differences from the mean first: x rstd - mean rstd would save an instruction, no
// time, and turn rows that are all alike into rounding errors times 1 / sqrt(eps).)
template <int W> struct Channels { float mean[W], rstd[W], w[W], b[W]; };
template <int V, int NC>
__device__ __forceinline__ void load_affine(const GnArgs& a, const Place<V>& p, int c0, Channels<V * NC>& k) {
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int cv = p.tx + GN_THREADS * j;
    if (NC > 1 && cv >= p.cols) break;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      k.w[V * j + c] = a.w ? a.w[c0 + cv * V + c] : 1.f;
      k.b[V * j + c] = a.b ? a.b[c0 + cv * V + c] : 0.f;
    }
  }
}
// of [mean, rstd] pairs of the segment, group by group
template <int V, int NC>
__device__ __forceinline__ void load_stats(const float* stats, const Place<V>& p, int c0, int cg, Channels<V * NC>& k) {
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int cv = p.tx + GN_THREADS * j;
    if (NC > 1 && cv >= p.cols) break;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const int g = (c0 + cv * V + c) / cg;
      k.mean[V * j + c] = stats[2 * g];
      k.rstd[V * j + c] = stats[2 * g + 1];
    }
  }
}

// y of [from, to) x [c0, c0 + width)
template <typename T, int V, int NC, bool ACT>
__device__ __forceinline__ void apply_rows(const GnArgs& a, const Place<V>& p, const Channels<V * NC>& k, int64_t from, int64_t to, int c0) {
  const int rows = thread_rows(p, from, to);
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int cv = p.tx + GN_THREADS * j;
    if (NC > 1 && cv >= p.cols) break;
    Stream<T, V> in(a.x, a.ld_x, p, from, c0 + cv * V), out(a.y, a.ld_y, p, from, c0 + cv * V);
    batches<GN_BATCH>(rows, [&](int count, auto whole) {
      Vec<T, V> v[GN_BATCH];
      in.read_last(v, count, whole);
#pragma unroll
      for (int i = 0; i < GN_BATCH; ++i) {
        if (!decltype(whole)::value && i >= count) break;
        float x[V];
        unpack(v[i], x);
        if constexpr (V == 1) {
          const float z = fmaf((x[0] - k.mean[j]) * k.rstd[j], k.w[j], k.b[j]);
          x[0] = ACT ? silu_fast_f(z) : z;
        } else {
#pragma unroll
          for (int c = 0; c < V; c += 2) {
            const f2 xh = less(two(x[c], x[c + 1]), two(k.mean[c], k.mean[c + 1])) * two(k.rstd[c], k.rstd[c + 1]);
            const f2 z = fma2(xh, two(k.w[c], k.w[c + 1]), two(k.b[c], k.b[c + 1]));
            apart(ACT ? silu_fast_2(z) : z, x[c], x[c + 1]);
          }
        }
        Vec<T, V> o;
        pack(x, o);
        out.write(o);
      }
    });
  }
}
template <typename T, int V, int NC>
__device__ __forceinline__ void zero_rows(void* out, int64_t ld, int channels, int64_t from, int64_t to) {
  const Place<V> p(channels);
  if (!p.used) return;
  T* const y = static_cast<T*>(out);
  for (int64_t r = from + p.ty; r < to; r += p.ty_n)
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int cv = p.tx + GN_THREADS * j;
      if (NC > 1 && cv >= p.cols) break;
      *reinterpret_cast<Vec<T, V>*>(y + r * ld + cv * V) = Vec<T, V>{};
    }
}
// Rows that belong to no segment (before the first, behind the last), shared out over `blocks` blocks
template <typename T, int V, int NC>
__device__ void zero_rest(const GnArgs& a, void* out, int64_t ld, int block, int blocks) {
  if (!a.seg_ptr) return;
  const int64_t head = min(max((int64_t)a.seg_ptr[0], (int64_t)0), a.n_rows);
  const int64_t tail = min(max((int64_t)a.seg_ptr[a.n_seg], head), a.n_rows);
  auto part = [&](int64_t from, int64_t to) {
    const int64_t n = to - from, per = (n + blocks - 1) / blocks;
    const int64_t f = from + per * block;
    if (f < to) zero_rows<T, V, NC>(out, ld, a.channels, f, min(f + per, to));
  };
  part(0, head);
  part(tail, a.n_rows);
}

__device__ __forceinline__ float rstd_of(float m2, float count, float eps) {
  return rsqrtf((count > 0.f ? m2 / count : 0.f) + eps);
}

template <typename T, int V, int NC, bool ACT>
__global__ void __launch_bounds__(GN_THREADS, gn_blocks(V, true)) k_group_norm(const __grid_constant__ GnArgs a) {
  pdl_sync();
  __shared__ GnShared<V * NC> sh;
  const int cg = a.channels / a.groups, slabs = a.groups / a.slab_groups, width = cg * a.slab_groups;
  const int64_t units = (int64_t)a.n_seg * slabs;
  if (blockIdx.x >= units) {
    zero_rest<T, V, NC>(a, a.y, a.ld_y, (int)(blockIdx.x - units), (int)(gridDim.x - units));
    return;
  }
  const int64_t s = blockIdx.x / slabs;
  const int c0 = (int)(blockIdx.x % slabs) * width;
  int64_t from, to;
  segment_rows(a, s, from, to);
  if (by_chunks(a, to - from)) return;
  block_stats<T, V, NC>(a, sh, from, to, c0, width, cg);
  float* const stats = a.stats + 2 * (s * a.groups + c0 / cg);
  const float count = (float)(to - from) * (float)cg;
  for (int g = threadIdx.x; g < a.slab_groups; g += GN_THREADS) {
    const float rstd = rstd_of(sh.group[1][g], count, a.eps);
    stats[2 * g] = sh.group[0][g];
    stats[2 * g + 1] = rstd;
    sh.group[1][g] = rstd;
  }
  __syncthreads();
  const Place<V> p(width);
  Channels<V * NC> k;
  load_affine<V, NC>(a, p, c0, k);
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int cv = p.tx + GN_THREADS * j;
    if (NC > 1 && cv >= p.cols) break;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const int g = (cv * V + c) / cg;
      k.mean[V * j + c] = sh.group[0][g];
      k.rstd[V * j + c] = sh.group[1][g];
    }
  }
  apply_rows<T, V, NC, ACT>(a, p, k, from, to, c0);
}

// ------------------------------------------------------------------ by chunks
// f(segment, its rows in the chunk) for every segment that goes by chunks and has rows in [c_from, c_to), in order
template <typename F> __device__ __forceinline__ void for_segments(const GnArgs& a, int64_t c_from, int64_t c_to, F f) {
  int64_t s = 0;
  if (a.seg_ptr) {  // the last segment that starts at or before c_from, or the first
    int64_t lo = 0, hi = a.n_seg;  // 32 probes at a time: two rounds for a thousand segments
    while (hi - lo > 1) {
      const int64_t step = (hi - lo + 31) / 32, at = lo + step * (threadIdx.x & 31);
      const unsigned below = __ballot_sync(0xffffffffu, at < hi && (int64_t)a.seg_ptr[at] <= c_from);
      // offsets are in order: the probes at or below c_from come first (whatever they hold, lo and hi close in)
      const int n = __popc(below);
      const int64_t next = n > 0 ? lo + step * (n - 1) : lo;
      hi = min(next + step, hi);
      lo = min(next, hi - 1);
    }
    s = lo;
  } else {
    s = c_from / (a.n_rows / a.n_seg);
  }
  for (; s < a.n_seg; ++s) {
    int64_t from, to;
    segment_rows(a, s, from, to);
    if (from >= c_to) break;
    const bool chunked = by_chunks(a, to - from);
    from = max(from, c_from);
    to = min(to, c_to);
    if (chunked && from < to) f(s, from, to);
  }
}

template <typename T, int V, int NC>
__global__ void __launch_bounds__(GN_THREADS, gn_blocks(V)) k_group_norm_part(const __grid_constant__ GnArgs a) {
  pdl_sync();
  __shared__ GnShared<V * NC> sh;
  const int cg = a.channels / a.groups;
  const int64_t c_from = (int64_t)blockIdx.x * a.chunk, c_to = min(c_from + a.chunk, a.n_rows);
  for_segments(a, c_from, c_to, [&](int64_t s, int64_t from, int64_t to) {
    block_stats<T, V, NC>(a, sh, from, to, 0, a.channels, cg);
    float* const part = a.part + 2 * ((int64_t)blockIdx.x + s) * a.groups;
    for (int g = threadIdx.x; g < a.groups; g += GN_THREADS) { part[2 * g] = sh.group[0][g]; part[2 * g + 1] = sh.group[1][g]; }
  });
}

// Warp per (segment, group): the chunks' statistics, each lane its chunks in order, then the lanes.  blockIdx.x = segment, the blocks of
// a segment take its groups in turn: most segments go by blocks, and theirs are gone after one look.
__global__ void __launch_bounds__(GN_THREADS) k_group_norm_join(const __grid_constant__ GnArgs a) {
  pdl_sync();
  const int64_t s = blockIdx.x;
  const int lane = threadIdx.x & 31, cg = a.channels / a.groups;
  int64_t from, to;
  segment_rows(a, s, from, to);
  if (!by_chunks(a, to - from)) return;
  for (int g = blockIdx.y * GN_WARPS + (threadIdx.x >> 5); g < a.groups; g += gridDim.y * GN_WARPS) {
    float n = 0.f, mean = 0.f, m2 = 0.f;
    if (from < to)
      for (int64_t c0 = from / a.chunk + lane; c0 <= (to - 1) / a.chunk; c0 += 32 * 8) {
        float2 v[8];  // eight chunks' loads in flight
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c0 + 32 * i <= (to - 1) / a.chunk) v[i] = *reinterpret_cast<const float2*>(a.part + 2 * ((c0 + 32 * i + s) * a.groups + g));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int64_t c = c0 + 32 * i, f = max(from, c * a.chunk), t = min(to, (c + 1) * a.chunk);
          if (f >= t) break;
          const float nb = (float)(t - f);
          join(n, mean, m2, nb, v[i].x, v[i].y / (float)cg);  // in units of rows: counts are exact up to 2^24, good to 2^-24 above
          n += nb;
        }
      }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float nb = __shfl_xor_sync(0xffffffffu, n, o), mo = __shfl_xor_sync(0xffffffffu, mean, o), so = __shfl_xor_sync(0xffffffffu, m2, o);
      const bool low_lane = (lane & o) == 0;
      float n1 = low_lane ? n : nb, m1 = low_lane ? mean : mo, s1 = low_lane ? m2 : so;
      join(n1, m1, s1, low_lane ? nb : n, low_lane ? mo : mean, low_lane ? so : m2);
      n += nb; mean = m1; m2 = s1;
    }
    if (lane == 0) {
      a.stats[2 * (s * a.groups + g)] = mean;
      a.stats[2 * (s * a.groups + g) + 1] = rstd_of(m2, n, a.eps);
    }
  }
}

template <typename T, int V, int NC, bool ACT>
__global__ void __launch_bounds__(GN_THREADS, gn_blocks(V)) k_group_norm_apply(const __grid_constant__ GnArgs a) {
  pdl_sync();
  const int64_t chunk = (int64_t)gridDim.x - 1 - blockIdx.x;  // the last chunks' rows are the ones still in L2
  const int64_t c_from = chunk * a.chunk, c_to = min(c_from + a.chunk, a.n_rows);
  const int cg = a.channels / a.groups;
  const Place<V> p(a.channels);
  Channels<V * NC> k;
  if (p.used) load_affine<V, NC>(a, p, 0, k);
  for_segments(a, c_from, c_to, [&](int64_t s, int64_t from, int64_t to) {
    if (p.used) load_stats<V, NC>(a.stats + 2 * s * a.groups, p, 0, cg, k);
    apply_rows<T, V, NC, ACT>(a, p, k, from, to, 0);
  });
  if (a.zero_rest) zero_rest<T, V, NC>(a, a.y, a.ld_y, (int)blockIdx.x, (int)gridDim.x);
}

// ------------------------------------------------------------------ backward
// Sums of dz and dz xh over [from, to), channel by channel, into sh.first[c], sh.second[c]
template <typename T, int V, int NC, bool ACT>
__device__ void block_sums(const GnArgs& a, GnShared<V * NC>& sh, const Place<V>& p, const Channels<V * NC>& k, int64_t from, int64_t to, int c0,
                           int width) {
  float s1[V * NC], s2[V * NC];
#pragma unroll
  for (int i = 0; i < V * NC; ++i) s1[i] = s2[i] = 0.f;
  const int rows = thread_rows(p, from, to);
  if (rows > 0) {
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int cv = p.tx + GN_THREADS * j;
      if (NC > 1 && cv >= p.cols) break;
      constexpr int U = gn_pairs<V>;
      Stream<T, V> in(a.x, a.ld_x, p, from, c0 + cv * V), grad(a.dy, a.ld_dy, p, from, c0 + cv * V);
      batches<U>(rows, [&](int count, auto whole) {
        Vec<T, V> v[U], d[U];
        in.read(v, count, whole);
        grad.read(d, count, whole);
#pragma unroll
        for (int i = 0; i < U; ++i) {
          if (!decltype(whole)::value && i >= count) break;
          float x[V], g[V];
          unpack(v[i], x);
          unpack(d[i], g);
          if constexpr (V == 1) {
            const float xh = (x[0] - k.mean[j]) * k.rstd[j];
            const float dz = ACT ? g[0] * silu_grad_fast_f(fmaf(xh, k.w[j], k.b[j])) : g[0];
            s1[j] += dz;
            s2[j] = fmaf(dz, xh, s2[j]);
          } else {
#pragma unroll
            for (int c = 0; c < V; c += 2) {
              const f2 xh = less(two(x[c], x[c + 1]), two(k.mean[c], k.mean[c + 1])) * two(k.rstd[c], k.rstd[c + 1]);
              f2 dz = two(g[c], g[c + 1]);
              if constexpr (ACT) dz = dz * silu_grad_fast_2(fma2(xh, two(k.w[c], k.w[c + 1]), two(k.b[c], k.b[c + 1])));
              apart(two(s1[c], s1[c + 1]) + dz, s1[c], s1[c + 1]);
              apart(fma2(dz, xh, two(s2[c], s2[c + 1])), s2[c], s2[c + 1]);
            }
          }
        }
      });
    }
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool fold = p.tx_n < 32 && (p.tx_n & (p.tx_n - 1)) == 0;
  if (fold)
    for (int o = p.tx_n; o < 32; o <<= 1)
#pragma unroll
      for (int i = 0; i < V * NC; ++i) {
        s1[i] += __shfl_xor_sync(0xffffffffu, s1[i], o);
        s2[i] += __shfl_xor_sync(0xffffffffu, s2[i], o);
      }
  const int entries = fold ? GN_WARPS : p.ty_n, e = fold ? warp : p.ty;
  __syncthreads();
  if (p.used && (!fold || lane < p.tx_n)) {
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int cv = p.tx + GN_THREADS * j;
      if (NC > 1 && cv >= p.cols) break;
#pragma unroll
      for (int c = 0; c < V; ++c) {
        sh.first[e * width + cv * V + c] = s1[V * j + c];
        sh.second[e * width + cv * V + c] = s2[V * j + c];
      }
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < width; c += GN_THREADS) {  // a channel's column is its thread's alone
    float t1 = 0.f, t2 = 0.f;
    for (int i = 0; i < entries; ++i) { t1 += sh.first[i * width + c]; t2 += sh.second[i * width + c]; }
    sh.first[c] = t1;
    sh.second[c] = t2;
  }
  __syncthreads();
}

// dx of [from, to) x [c0, c0 + width); m1, m2: the groups' means of g and g xh
template <typename T, int V, int NC, bool ACT>
__device__ __forceinline__ void gradient_rows(const GnArgs& a, const Place<V>& p, const Channels<V * NC>& k, const float (&m1)[V * NC],
                                              const float (&m2)[V * NC], int64_t from, int64_t to, int c0) {
  const int rows = thread_rows(p, from, to);
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int cv = p.tx + GN_THREADS * j;
    if (NC > 1 && cv >= p.cols) break;
    constexpr int U = gn_pairs<V>;
    Stream<T, V> in(a.x, a.ld_x, p, from, c0 + cv * V), grad(a.dy, a.ld_dy, p, from, c0 + cv * V), out(a.dx, a.ld_dx, p, from, c0 + cv * V);
    batches<U>(rows, [&](int count, auto whole) {
      Vec<T, V> v[U], d[U];
      in.read_last(v, count, whole);
      grad.read_last(d, count, whole);
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (!decltype(whole)::value && i >= count) break;
        float x[V], g[V];
        unpack(v[i], x);
        unpack(d[i], g);
        if constexpr (V == 1) {
          const float xh = (x[0] - k.mean[j]) * k.rstd[j];
          const float dz = ACT ? g[0] * silu_grad_fast_f(fmaf(xh, k.w[j], k.b[j])) : g[0];
          x[0] = k.rstd[j] * (fmaf(dz, k.w[j], -m1[j]) - xh * m2[j]);
        } else {
#pragma unroll
          for (int c = 0; c < V; c += 2) {
            const f2 xh = less(two(x[c], x[c + 1]), two(k.mean[c], k.mean[c + 1])) * two(k.rstd[c], k.rstd[c + 1]), w = two(k.w[c], k.w[c + 1]);
            f2 dz = two(g[c], g[c + 1]);
            if constexpr (ACT) dz = dz * silu_grad_fast_2(fma2(xh, w, two(k.b[c], k.b[c + 1])));
            const f2 rest = fma2(xh, two(m2[c], m2[c + 1]), two(m1[c], m1[c + 1]));
            apart(two(k.rstd[c], k.rstd[c + 1]) * less(dz * w, rest), x[c], x[c + 1]);
          }
        }
        Vec<T, V> o;
        pack(x, o);
        out.write(o);
      }
    });
  }
}

// the groups' means from a slab's channel sums: sh.group[0 / 1][group of the slab]
template <int W>
__device__ __forceinline__ void group_means(const GnArgs& a, GnShared<W>& sh, const float* first, const float* second, int stride, int c0, int width,
                                            int cg, float count) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int g = warp; g < width / cg; g += GN_WARPS) {
    float t1 = 0.f, t2 = 0.f;
    for (int i = lane; i < cg; i += 32) {
      const int c = g * cg + i;
      const float w = a.w ? a.w[c0 + c] : 1.f;
      t1 = fmaf(w, first[c * stride], t1);
      t2 = fmaf(w, second[c * stride], t2);
    }
    t1 = warp_sum(t1);
    t2 = warp_sum(t2);
    if (lane == 0) {
      sh.group[0][g] = count > 0.f ? t1 / count : 0.f;
      sh.group[1][g] = count > 0.f ? t2 / count : 0.f;
    }
  }
  __syncthreads();
}
template <int V, int NC>
__device__ __forceinline__ void load_means(const GnShared<V * NC>& sh, const Place<V>& p, int cg, float (&m1)[V * NC], float (&m2)[V * NC]) {
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int cv = p.tx + GN_THREADS * j;
    if (NC > 1 && cv >= p.cols) break;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const int g = (cv * V + c) / cg;
      m1[V * j + c] = sh.group[0][g];
      m2[V * j + c] = sh.group[1][g];
    }
  }
}

template <typename T, int V, int NC, bool ACT>
__global__ void __launch_bounds__(GN_THREADS, gn_blocks(V)) k_group_norm_bwd(const __grid_constant__ GnArgs a) {
  pdl_sync();
  __shared__ GnShared<V * NC> sh;
  const int cg = a.channels / a.groups, slabs = a.groups / a.slab_groups, width = cg * a.slab_groups;
  const int64_t units = (int64_t)a.n_seg * slabs;
  if (blockIdx.x >= units) {
    zero_rest<T, V, NC>(a, a.dx, a.ld_dx, (int)(blockIdx.x - units), (int)(gridDim.x - units));
    return;
  }
  const int64_t s = blockIdx.x / slabs;
  const int c0 = (int)(blockIdx.x % slabs) * width;
  int64_t from, to;
  segment_rows(a, s, from, to);
  if (by_chunks(a, to - from)) return;
  const Place<V> p(width);
  Channels<V * NC> k;
  load_affine<V, NC>(a, p, c0, k);
  load_stats<V, NC>(a.stats + 2 * s * a.groups, p, c0, cg, k);
  block_sums<T, V, NC, ACT>(a, sh, p, k, from, to, c0, width);
  for (int c = threadIdx.x; c < width; c += GN_THREADS) {
    float* const sums = a.sums + 2 * (s * a.channels + c0 + c);
    sums[0] = sh.first[c];
    sums[1] = sh.second[c];
  }
  group_means(a, sh, sh.first, sh.second, 1, c0, width, cg, (float)(to - from) * (float)cg);
  float m1[V * NC], m2[V * NC];
  load_means<V, NC>(sh, p, cg, m1, m2);
  gradient_rows<T, V, NC, ACT>(a, p, k, m1, m2, from, to, c0);
}

template <typename T, int V, int NC, bool ACT>
__global__ void __launch_bounds__(GN_THREADS, gn_blocks(V)) k_group_norm_bwd_part(const __grid_constant__ GnArgs a) {
  pdl_sync();
  __shared__ GnShared<V * NC> sh;
  const int cg = a.channels / a.groups;
  const int64_t c_from = (int64_t)blockIdx.x * a.chunk, c_to = min(c_from + a.chunk, a.n_rows);
  const Place<V> p(a.channels);
  Channels<V * NC> k;
  load_affine<V, NC>(a, p, 0, k);
  for_segments(a, c_from, c_to, [&](int64_t s, int64_t from, int64_t to) {
    load_stats<V, NC>(a.stats + 2 * s * a.groups, p, 0, cg, k);
    block_sums<T, V, NC, ACT>(a, sh, p, k, from, to, 0, a.channels);
    float* const part = a.part + 2 * ((int64_t)blockIdx.x + s) * a.channels;
    for (int c = threadIdx.x; c < a.channels; c += GN_THREADS) { part[2 * c] = sh.first[c]; part[2 * c + 1] = sh.second[c]; }
  });
}

// the same for the channels' sums
__global__ void __launch_bounds__(GN_THREADS) k_group_norm_bwd_join(const __grid_constant__ GnArgs a) {
  pdl_sync();
  const int64_t s = blockIdx.x;
  const int lane = threadIdx.x & 31;
  int64_t from, to;
  segment_rows(a, s, from, to);
  if (!by_chunks(a, to - from)) return;
  for (int c = blockIdx.y * GN_WARPS + (threadIdx.x >> 5); c < a.channels; c += gridDim.y * GN_WARPS) {
    float t1 = 0.f, t2 = 0.f;
    if (from < to)
      for (int64_t c0 = from / a.chunk + lane; c0 <= (to - 1) / a.chunk; c0 += 32 * 8) {
        float2 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          v[i] = c0 + 32 * i <= (to - 1) / a.chunk ? *reinterpret_cast<const float2*>(a.part + 2 * ((c0 + 32 * i + s) * a.channels + c))
                                                   : make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 8; ++i) { t1 += v[i].x; t2 += v[i].y; }
      }
    t1 = warp_sum(t1);
    t2 = warp_sum(t2);
    if (lane == 0) { a.sums[2 * (s * a.channels + c)] = t1; a.sums[2 * (s * a.channels + c) + 1] = t2; }
  }
}

template <typename T, int V, int NC, bool ACT>
__global__ void __launch_bounds__(GN_THREADS, gn_blocks(V)) k_group_norm_bwd_apply(const __grid_constant__ GnArgs a) {
  pdl_sync();
  __shared__ GnShared<V * NC> sh;
  const int64_t chunk = (int64_t)gridDim.x - 1 - blockIdx.x;
  const int64_t c_from = chunk * a.chunk, c_to = min(c_from + a.chunk, a.n_rows);
  const int cg = a.channels / a.groups;
  const Place<V> p(a.channels);
  Channels<V * NC> k;
  load_affine<V, NC>(a, p, 0, k);
  for_segments(a, c_from, c_to, [&](int64_t s, int64_t from, int64_t to) {
    int64_t all_from, all_to;
    segment_rows(a, s, all_from, all_to);
    load_stats<V, NC>(a.stats + 2 * s * a.groups, p, 0, cg, k);
    const float* const sums = a.sums + 2 * s * a.channels;
    __syncthreads();  // the previous segment's means have been read
    group_means(a, sh, sums, sums + 1, 2, 0, a.channels, cg, (float)(all_to - all_from) * (float)cg);
    float m1[V * NC], m2[V * NC];
    load_means<V, NC>(sh, p, cg, m1, m2);
    gradient_rows<T, V, NC, ACT>(a, p, k, m1, m2, from, to, 0);
  });
  if (a.zero_rest) zero_rest<T, V, NC>(a, a.dx, a.ld_dx, (int)blockIdx.x, (int)gridDim.x);
}

// dw, db: a block takes 32 channels, its 32 warps the segments in turn, eight loads in flight; 64-bit sums (a few KB, and segments may
// be many)
constexpr int GN_AFFINE_THREADS = 1024;
__global__ void __launch_bounds__(GN_AFFINE_THREADS) k_group_norm_affine(const __grid_constant__ GnArgs a, float* __restrict__ dw,
                                                                         float* __restrict__ db) {
  pdl_sync();
  constexpr int WARPS = GN_AFFINE_THREADS / 32;
  __shared__ double sh[WARPS][2][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane;
  double t1 = 0., t2 = 0.;
  if (c < a.channels)
    for (int64_t s0 = warp; s0 < a.n_seg; s0 += 8 * WARPS) {
      float2 v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t s = s0 + i * WARPS;
        v[i] = s < a.n_seg ? *reinterpret_cast<const float2*>(a.sums + 2 * (s * a.channels + c)) : make_float2(0.f, 0.f);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) { t1 += (double)v[i].x; t2 += (double)v[i].y; }
    }
  sh[warp][0][lane] = t1;
  sh[warp][1][lane] = t2;
  __syncthreads();
  if (warp < 2 && c < a.channels) {
    double t = 0.;
#pragma unroll 8
    for (int i = 0; i < WARPS; ++i) t += sh[i][warp][lane];
    float* const out = warp == 0 ? db : dw;
    if (out) out[c] = (float)t;
  }
}

// ------------------------------------------------------------------ host side
static bool gn_valid(const mb_group_norm* d) {
  if (!d || d->n_rows < 0 || d->n_seg < 0 || d->channels < 1 || d->channels > GN_MAX_CHANNELS || d->groups < 1) return false;
  if (d->channels % d->groups || d->dtype < 0 || d->dtype > 2 || d->act < 0 || d->act > 1 || !(d->eps > 0.f)) return false;
  if (!d->seg_ptr && d->n_seg > 0 && d->n_rows % d->n_seg) return false;
  if (reinterpret_cast<uintptr_t>(d->scratch) & 15u) return false;
  return d->n_rows <= INT32_MAX;
}
// Rows of a chunk: as many as put one block into each of GN_PLACES places of every multiprocessor, so that they all run at once.  (Every chunk
// costs its block some 2 us beside the rows: 409,601 bf16 rows of 256 in chunks of 128 take 206 us, of 512 163, of 1,384 140.)
static int gn_chunk(int64_t n_rows, int n_sm) {
  const int64_t r = (n_rows + GN_PLACES * n_sm - 1) / (GN_PLACES * n_sm);
  return (int)(r < 32 ? 32 : (r + 7) / 8 * 8);
}
// Longest segment that a block takes (slab by slab), -1: none.  Few rows: all of them, three launches fewer.  Segments that are long on
// average: none.  Forward, float32 rows of 128 in eight groups, even segments, by blocks / by chunks:
//     1,024 rows of one segment 14.3 / 14.3 us, of eight 8.2 / 13.8;      2,048 rows of one 20.5 / 13.8;     8,192 of eight 14.3 / 16.4
//     16,384 rows of four segments 32.8 / 20.5, of eight 22.5 / 19.9, of sixteen 14.4 / 20.5
//     573,894 rows of 128 segments 166 / 160, of 280 135 / 160, of 512 123 / 160 (131 as it is: launches that find no long segment)
// The line goes by the average: one long segment among short ones is left to a few blocks (15,000 of 16,000 rows 96 us, by chunks 23).
static int gn_limit(int64_t n_rows, int n_seg) {
  if (n_rows <= 1024) return 1024;
  if (n_rows > 2048 * (int64_t)n_seg) return -1;
  return n_rows <= 16384 ? 16384 : 4096;
}
static int gn_prepare(const mb_group_norm* d, GnArgs& a, int& n_sm) {
  int rc = sm_count(&n_sm);
  if (rc) return rc;
  a = GnArgs{};
  a.n_rows = d->n_rows; a.ld_x = d->ld_x; a.ld_y = d->ld_y; a.ld_dy = d->ld_dy; a.ld_dx = d->ld_dx;
  a.seg_ptr = d->seg_ptr; a.n_seg = d->n_seg; a.channels = d->channels; a.groups = d->groups; a.act = d->act; a.zero_rest = d->zero_rest;
  a.eps = d->eps; a.x = d->x; a.dy = d->dy; a.w = d->weight; a.b = d->bias; a.y = d->y; a.dx = d->dx; a.stats = d->stats;
  a.chunk = gn_chunk(d->n_rows, n_sm);
  a.limit = gn_limit(d->n_rows, d->n_seg);
  return MB_OK;
}
static bool gn_vector(const mb_group_norm* d, std::initializer_list<const void*> rows, std::initializer_list<int64_t> lds) {
  const int size = d->dtype == MB_DTYPE_F32 ? 4 : 2, v = 16 / size;
  if (d->channels % v) return false;
  for (const void* p : rows) if (reinterpret_cast<uintptr_t>(p) & 15u) return false;
  for (int64_t ld : lds) if (ld % v) return false;
  return true;
}
// Groups of a slab: as few as give 128 bytes of a row and, segments being short, some 16 KB of a segment; whole vectors, slabs of one
// size.  (256 segments of 36 rows of 512 bytes: 29 us by slabs of 64 bytes, 20 of 128, 11 whole.)
static int gn_slab(const mb_group_norm* d, int v) {
  const int64_t size = d->dtype == MB_DTYPE_F32 ? 4 : 2, cg = d->channels / d->groups, average = d->n_rows / d->n_seg + 1;
  const int64_t least = average < 128 ? 16384 / average : 128;
  for (int g = 1; g < d->groups; ++g)
    if (d->groups % g == 0 && (g * cg) % v == 0 && g * cg * size >= least && g * cg / v <= GN_THREADS) return g;
  return d->groups;
}
template <typename F> static void gn_typed(int dtype, bool vec, F f) {
  if (dtype == MB_DTYPE_F32) { if (vec) f.template operator()<float, 4, 1>(); else f.template operator()<float, 1, 4>(); }
  else if (dtype == MB_DTYPE_BF16) { if (vec) f.template operator()<__nv_bfloat16, 8, 1>(); else f.template operator()<__nv_bfloat16, 1, 4>(); }
  else { if (vec) f.template operator()<__half, 8, 1>(); else f.template operator()<__half, 1, 4>(); }
}
static dim3 gn_join_grid(int n_seg, int units) {  // some 1,024 blocks, a warp for every unit of one segment at the most
  const int all = cdiv(units, GN_WARPS), want = 1024 / n_seg;
  return dim3((unsigned)n_seg, (unsigned)(want < 1 ? 1 : want < all ? want : all));
}
struct GnFwdLaunch {
  const GnArgs& a; int n_sm; cudaStream_t st; bool blocks, chunks;
  template <typename T, int V, int NC> void operator()() const {
    const int slabs = a.groups / a.slab_groups;
    if (blocks) {
      const int rest = a.zero_rest && a.seg_ptr && !chunks ? (int)(a.n_rows / 256 < n_sm ? a.n_rows / 256 + 1 : n_sm) : 0;
      const unsigned grid = (unsigned)(a.n_seg * slabs + rest);
      if (a.act) launch(k_group_norm<T, V, NC, true>, grid, GN_THREADS, 0, st, a);
      else launch(k_group_norm<T, V, NC, false>, grid, GN_THREADS, 0, st, a);
    }
    if (chunks) {
      const unsigned grid = (unsigned)cdiv(a.n_rows, a.chunk);
      launch(k_group_norm_part<T, V, NC>, grid, GN_THREADS, 0, st, a);
      launch(k_group_norm_join, gn_join_grid(a.n_seg, a.groups), GN_THREADS, 0, st, a);
      if (a.act) launch(k_group_norm_apply<T, V, NC, true>, grid, GN_THREADS, 0, st, a);
      else launch(k_group_norm_apply<T, V, NC, false>, grid, GN_THREADS, 0, st, a);
    }
  }
};
struct GnBwdLaunch {
  const GnArgs& a; int n_sm; cudaStream_t st; bool blocks, chunks;
  template <typename T, int V, int NC> void operator()() const {
    if (a.act) go<T, V, NC, true>(); else go<T, V, NC, false>();
  }
  template <typename T, int V, int NC, bool ACT> void go() const {
    const int slabs = a.groups / a.slab_groups;
    if (blocks) {
      const int rest = a.zero_rest && a.seg_ptr && !chunks ? (int)(a.n_rows / 256 < n_sm ? a.n_rows / 256 + 1 : n_sm) : 0;
      launch(k_group_norm_bwd<T, V, NC, ACT>, (unsigned)(a.n_seg * slabs + rest), GN_THREADS, 0, st, a);
    }
    if (chunks) {
      const unsigned grid = (unsigned)cdiv(a.n_rows, a.chunk);
      launch(k_group_norm_bwd_part<T, V, NC, ACT>, grid, GN_THREADS, 0, st, a);
      launch(k_group_norm_bwd_join, gn_join_grid(a.n_seg, a.channels), GN_THREADS, 0, st, a);
      launch(k_group_norm_bwd_apply<T, V, NC, ACT>, grid, GN_THREADS, 0, st, a);
    }
  }
};

}  // namespace mb

using namespace mb;

extern "C" size_t mb_group_norm_scratch(int64_t n_rows, int32_t n_seg, int32_t channels, int32_t backward) {
  // backward: the segments' sums; with segments that go by chunks: their partial results, rows chunk + segment
  int n_sm = 0;
  if (n_rows < 0 || n_seg < 0 || channels < 1 || sm_count(&n_sm) != MB_OK) return 0;
  const int64_t limit = gn_limit(n_rows, n_seg), r = gn_chunk(n_rows, n_sm);
  const int64_t part = limit < 0 || n_rows > limit ? (n_rows + r - 1) / r + n_seg : 0;
  return 2 * sizeof(float) * (size_t)channels * (size_t)(part + (backward ? n_seg : 0));
}

extern "C" int mb_group_norm_fwd(const mb_group_norm* d, void* stream) {
  if (!gn_valid(d) || (d->n_rows > 0 && (!d->x || !d->y || d->ld_x < d->channels || d->ld_y < d->channels))) return MB_ERR_INVALID;
  if (d->n_seg > 0 && !d->stats) return MB_ERR_INVALID;
  if (d->n_seg == 0 || d->n_rows == 0) return MB_OK;
  GnArgs a;
  int n_sm = 0, rc = gn_prepare(d, a, n_sm);
  if (rc) return rc;
  if (!d->scratch && (a.limit < 0 || a.n_rows > a.limit)) return MB_ERR_INVALID;
  const bool vec = gn_vector(d, {d->x, d->y}, {d->ld_x, d->ld_y});
  a.slab_groups = gn_slab(d, vec ? (d->dtype == MB_DTYPE_F32 ? 4 : 8) : 1);
  if ((int64_t)a.n_seg * (a.groups / a.slab_groups) + n_sm > INT32_MAX) return MB_ERR_OVERFLOW;
  a.part = static_cast<float*>(d->scratch);
  gn_typed(d->dtype, vec, GnFwdLaunch{a, n_sm, (cudaStream_t)stream, a.limit >= 0, a.limit < 0 || a.n_rows > a.limit});
  MB_LAUNCH_CHECK("k_group_norm");
  return MB_OK;
}

extern "C" int mb_group_norm_bwd(const mb_group_norm* d, void* stream) {
  if (!gn_valid(d) || (d->n_rows > 0 && (!d->x || !d->dy || !d->dx || d->ld_x < d->channels || d->ld_dy < d->channels || d->ld_dx < d->channels)))
    return MB_ERR_INVALID;
  if (d->n_seg > 0 && (!d->stats || !d->scratch)) return MB_ERR_INVALID;
  GnArgs a;
  int n_sm = 0, rc = gn_prepare(d, a, n_sm);
  if (rc) return rc;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool some = d->n_seg > 0 && d->n_rows > 0;
  if (some) {
    const bool vec = gn_vector(d, {d->x, d->dy, d->dx}, {d->ld_x, d->ld_dy, d->ld_dx});
    a.slab_groups = gn_slab(d, vec ? (d->dtype == MB_DTYPE_F32 ? 4 : 8) : 1);
    if ((int64_t)a.n_seg * (a.groups / a.slab_groups) + n_sm > INT32_MAX || (int64_t)a.n_seg * a.channels > INT32_MAX) return MB_ERR_OVERFLOW;
    a.sums = static_cast<float*>(d->scratch);
    a.part = a.sums + 2 * (size_t)a.n_seg * a.channels;
    gn_typed(d->dtype, vec, GnBwdLaunch{a, n_sm, st, a.limit >= 0, a.limit < 0 || a.n_rows > a.limit});
    MB_LAUNCH_CHECK("k_group_norm_bwd");
  } else {
    a.n_seg = 0;
  }
  if (d->dweight || d->dbias) {
    launch(k_group_norm_affine, (unsigned)cdiv(a.channels, 32), GN_AFFINE_THREADS, 0, st, a, d->dweight, d->dbias);
    MB_LAUNCH_CHECK("k_group_norm_affine");
  }
  return MB_OK;
}
