// Dense layers of a mixture of experts on rows grouped by expert: forward and data gradient (one product), weight gradient.
// (Included by gemm.cu inside namespace mb, after its tensor-core helpers and k_gemm_ps.)

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

// ------------------------------------------------------------------ forward and data gradient
// y[s] = act(f(x[idx[s]]) W_e^T + b_e) on the tensor cores: the roles of k_gemm_ps (which see) on row tiles that belong to one expert each.
//
// Row tiles are numbered through the experts, ceil(slots / 128) of them each; a warp finds a tile's expert with one scan over 32
// experts' counts at a time (Walk), from the offsets on the device, so that the host never reads them.  A tile's rows are gathered
// through idx, its weights are rows e n_out + 128 j .. of one tensor map over all experts' weights.  Rows behind the expert's last slot
// repeat it and are not stored: the next expert's rows belong to another tile.
//
// Operands are split into two tf32 parts, hi rounded to nearest: x = hi + lo to 2^-22, and the three products kept drop lo lo, at
// most 2^-24 of |x w| and of either sign: the float32 rounding of the sums is as large.  (Two bf16 parts, as the other dense
// layers have, issue at twice the rate and are good to 2^-17.)
//
// 573,894 slots of 286,947 rows, 32 experts: 256 -> 128 in 230 us (163 TFLOP/s), 128 -> 256 in 268 (140).  Neither memory (90 and 135 us)
// nor the tensor cores (115 us at their tf32 rate) set that: an instruction takes the warp that issues it some 50 cycles, twelve a chunk,
// and a column block's accumulators are read out before the next block may use them.  One accumulator for both kinds of products, two of
// them in turn, took 180 and 186 us and lost 1.1e-6 / 1.8e-6 of the result's norm with 128 / 256 terms where this loses 4e-7 / 9e-7; two
// issuing warps, one for each kind, or sixteen epilogue warps 231 - 281 us.
//
// shared (K = 128): the four A buffers hold the whole row tile, converted once for all its column blocks.  Otherwise a column block is a
// tile of its own and its rows are gathered again, from L2.
#define MB_TMEM_LD16(taddr, v)                                                                                   \
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "                                                         \
               "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"                  \
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), \
                 "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]),        \
                 "=r"(v[15]) : "r"(taddr) : "memory")
struct alignas(64) ExMaps { CUtensorMap hi, lo; };

// Whether a phase is over, without waiting for it
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// The products of K steps [from, to) of a chunk (four of them): A in tensor memory at ta (hi | lo), weight or column tiles at wb (hi | lo).
// The large ones, hi hi, and the corrections, lo hi + hi lo, 2^-11 of them, have accumulators of their own: the tensor cores cut every sum
// to float32, towards zero, and a correction added to a large sum costs as much of it as another product.
__device__ __forceinline__ void large_products(uint32_t d_tmem, uint32_t ta, uint32_t wb, int from, int to, bool fresh) {
  const uint64_t dbh = umma_desc(wb);
#pragma unroll
  for (int kk = from; kk < to; ++kk) umma_tf32_ts(d_tmem, ta + 8 * kk, dbh + (uint64_t)(2 * kk), (!fresh || kk > 0) ? 1u : 0u);
}
__device__ __forceinline__ void small_products(uint32_t d_tmem, uint32_t ta, uint32_t wb, int from, int to, bool fresh) {
  const uint64_t dbh = umma_desc(wb), dbl = umma_desc(wb + TC_TILE_BYTES);
#pragma unroll
  for (int kk = from; kk < to; ++kk) {
    const uint64_t adv = (uint64_t)(2 * kk);
    umma_tf32_ts(d_tmem, ta + 32 + 8 * kk, dbh + adv, (!fresh || kk > 0) ? 1u : 0u);
    umma_tf32_ts(d_tmem, ta + 8 * kk, dbl + adv, 1u);
  }
}

// Tiles of 2^SHIFT slots in order of expert; all lanes of a warp call it together
template <int SHIFT> struct Walk {
  const mb_experts* d;
  int base, before, total;   // first expert held (lane l: base + l), tiles ahead of it, tiles of the 32
  int64_t from, to;
  int upto;                  // tiles of this and the lower lanes' experts
  __device__ __forceinline__ void load() {
    const int lane = threadIdx.x & 31, e = base + lane;
    from = to = 0;
    if (e < d->n_experts) expert_slots(*d, e, from, to);
    upto = (int)((to - from + (1 << SHIFT) - 1) >> SHIFT);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += u;
    }
    total = __shfl_sync(0xffffffffu, upto, 31);
  }
  __device__ __forceinline__ void start(const mb_experts& args) { d = &args; base = before = 0; load(); }
  // tile t (never less than the last one asked for): its expert, first slot, the expert's slots from there on and whether it is the
  // expert's first tile; false: there are no more
  __device__ __forceinline__ bool seek(int t, int& e, int64_t& s0, int64_t& left, bool& first) {
    while (t - before >= total) {
      before += total;
      base += 32;
      if (base >= d->n_experts) { total = before = 0; return false; }
      load();
    }
    const int at = __popc(__ballot_sync(0xffffffffu, t - before >= upto));
    const int ahead = __shfl_sync(0xffffffffu, upto, at > 0 ? at - 1 : 0), nth = t - before - (at > 0 ? ahead : 0);
    e = base + at;
    s0 = __shfl_sync(0xffffffffu, from, at) + ((int64_t)nth << SHIFT);
    left = __shfl_sync(0xffffffffu, to, at) - s0;
    first = nth == 0;
    return true;
  }
  __device__ __forceinline__ bool seek(int t, int& e, int64_t& s0, int& rows) {
    int64_t left;
    bool first;
    if (!seek(t, e, s0, left, first)) return false;
    rows = left < (1 << SHIFT) ? (int)left : 1 << SHIFT;
    return true;
  }
  // the tile after the one that (e, s0, left) describes, number t: without a search while the expert lasts
  __device__ __forceinline__ bool next(int t, int& e, int64_t& s0, int64_t& left, bool& first) {
    if (left > (1 << SHIFT)) {
      s0 += 1 << SHIFT;
      left -= 1 << SHIFT;
      first = false;
      return true;
    }
    return seek(t, e, s0, left, first);
  }
  // all tiles; the walk is at the start again
  __device__ __forceinline__ int64_t count() {
    int64_t n = 0;
    for (int b = 0; b < d->n_experts; b += 32) { base = b; load(); n += total; }
    base = before = 0;
    load();
    return n;
  }
};

// A producer warp spends some 2,500 cycles on a chunk of 32 x 32 values, most of them waiting for its own instructions, where the chunk's
// products take 768: sixteen of them, each chunk of four to a set of its own.
constexpr int EX_SETS = 4, EX_PROD_WARPS = 4 * EX_SETS, EX_EPI_WARP0 = PS_PROD_WARP0 + EX_PROD_WARPS, EX_THREADS = 32 * (EX_EPI_WARP0 + 8);
// Chunks whose products go into the accumulators before these are read: with more than 256 values of K a row's sum is joined from such runs
// in the epilogue, rounded to nearest, by way of the output (512 values in one run lost 1.4e-6 of the result's norm).
constexpr int EX_RUN = 8;
constexpr int EX_STAGES = 2;                                     // patches of a producer warp
constexpr int EX_W_SLOTS = 3;                                    // weight tiles (hi and lo) in flight
constexpr int EX_PATCH_OFF = EX_W_SLOTS * 2 * TC_TILE_BYTES;
constexpr int EX_BAR_OFF = EX_PATCH_OFF + EX_PROD_WARPS * EX_STAGES * 32 * 128;
constexpr int EX_BIAS_OFF = EX_BAR_OFF + 256;                    // an epilogue warp's 64 values of the bias
constexpr int EX_SMEM_BYTES = EX_BIAS_OFF + 8 * 256;
static_assert(EX_SMEM_BYTES <= 227 * 1024, "shared memory of one CTA");

// x = hi + lo, hi rounded to 11 significant bits by integer arithmetic (the conversion instruction runs at an eighth of the rate: two of
// them a value took 512 cycles of the 768 that a chunk's products need).  The tensor cores read lo's leading 11 bits, of |lo| <= 2^-12 |x|.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}
// Eight values; `seen` gathers their lo: no longer finite once hi has been rounded out of the finite numbers, at half an instruction a value.
__device__ __forceinline__ void split_tf32_all(const float (&x)[8], uint32_t (&hi)[8], uint32_t (&lo)[8], f2& seen) {
#pragma unroll
  for (int i = 0; i < 8; ++i) split_tf32(x[i], hi[i], lo[i]);
#pragma unroll
  for (int i = 0; i < 8; i += 2) seen = seen + two(__uint_as_float(lo[i]), __uint_as_float(lo[i + 1]));
}
// Whether any lane of the warp has to split its chunk again by split_tf32_large.  (The weight gradient of 573,894 slots, 256 -> 128: 298 us
// without the look, 308 so, 341 with a look at every eight values.)
__device__ __forceinline__ bool split_again(f2 seen) {
  float a, b;
  apart(seen, a, b);
  return __any_sync(0xffffffffu, !(fabsf(a + b) <= FLT_MAX));
}
// Next to 2^128 a finite x is cut instead of rounded; an infinity is left to lo, whose one product kept, with the other operand's hi, has
// the right sign.  (As hi it would meet the other operand's lo too, which is of either sign or zero: NaN.)
__device__ __forceinline__ void split_tf32_large(const float (&x)[8], uint32_t (&hi)[8], uint32_t (&lo)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = __float_as_uint(x[i]), size = u & 0x7FFFFFFFu;
    if (size < 0x7F7FF000u) split_tf32(x[i], hi[i], lo[i]);
    else {
      hi[i] = size < 0x7F800000u ? u & 0xFFFFE000u : 0u;
      lo[i] = __float_as_uint(x[i] - __uint_as_float(hi[i]));
    }
  }
}

__global__ void __launch_bounds__(EX_THREADS, 1) k_experts(const __grid_constant__ mb_experts d, const __grid_constant__ ExMaps maps, const int shared) {
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + EX_BAR_OFF);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + EX_BAR_OFF + 240);
  if ((smem_u32(smem) & 1023u) != 0) {  // the swizzled tiles need a 1024-byte aligned base
    if (threadIdx.x == 0) atomicOr(&g_gemm_status, 2);
    return;
  }
  // a_ready[4] (4 producer warps) a_done[4] | w_ready[3] w_done[3] | d_full d_free (8 epilogue warps) | retired
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t a_ready = bar0, a_done = bar0 + 32, w_ready = bar0 + 64, w_done = bar0 + 96, d_full = bar0 + 128, d_free = bar0 + 136,
                 retired = bar0 + 144;
  const uint32_t ring = smem_u32(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nb = d.n_out / 128, nch = d.n_in / TC_BK;
  const int per_tile = shared ? 1 : nb;      // items of a row tile; an item is a row tile, or one of its column blocks
  const int per_item = shared ? nb : 1;      // column blocks of an item

  if (warp == PS_MMA_WARP) {
    if (lane == 0) {
      for (int b = 0; b < 4; ++b) { mbar_init(a_ready + 8 * b, 4); mbar_init(a_done + 8 * b, 1); }
      for (int b = 0; b < EX_W_SLOTS; ++b) { mbar_init(w_ready + 8 * b, 1); mbar_init(w_done + 8 * b, 1); }
      mbar_init(d_full, 1);
      mbar_init(d_free, 8);
      mbar_init(retired, 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 :: "r"(smem_u32(tmem_slot)), "r"(PS_TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = *tmem_slot;
  pdl_sync();
  Walk<7> walk;
  walk.start(d);
  int e, rows;
  int64_t s0;

  if (warp == PS_MMA_WARP) {
    uint32_t elected;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(elected));
    const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem_base, 0), ring_u = __shfl_sync(0xffffffffu, ring, 0);
    // the number of this CTA's items, from one lane: the loop, and with it every operand of a matrix instruction, is the same for all lanes
    // by construction
    const int64_t items = walk.count() * per_tile;
    const int n_items = __shfl_sync(0xffffffffu, (int)((items - blockIdx.x + gridDim.x - 1) / gridDim.x), 0);
    bool alive = true;
    uint32_t g = 0, run = 0, slot = 0, phase = 0;  // A chunks and uses of the accumulators so far; weight slot and its use
    // The tensor cores' queue is a few instructions deep: issuing a chunk's twelve takes as long as they do, and then a wait that finds its
    // barrier open still takes 110 - 140 cycles, three of them a chunk.  So the next chunk's barriers are tested between this one's
    // instructions, and waited for only where that fails.
    bool open = false;
    for (int it = 0; it < n_items; ++it) {
      for (int j = 0; j < per_item; ++j) {
        for (int c = 0; c < nch; ++c) {
          const uint32_t ga = g + c, ab = ga & 3;
          if (!open) {
            if (j == 0 && alive) alive = mbar_wait(a_ready + 8 * ab, (ga >> 2) & 1);
            if (alive) alive = mbar_wait(w_ready + 8 * slot, phase & 1);
            if (c % EX_RUN == 0 && run >= 1 && alive) alive = mbar_wait(d_free, (run - 1) & 1);
            alive = __all_sync(0xffffffffu, alive);
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t ta = tmem_u + 256 + 64 * ab, wb = ring_u + slot * 2 * TC_TILE_BYTES;
          const uint32_t slot1 = slot + 1 == EX_W_SLOTS ? 0 : slot + 1, phase1 = slot1 == 0 ? phase + 1 : phase;
          const bool run_ends = c == nch - 1 || c % EX_RUN == EX_RUN - 1;
          const uint32_t g1 = ga + 1;
          if (elected) large_products(tmem_u, ta, wb, 0, 4, c % EX_RUN == 0);
          __syncwarp();
          bool ok = !run_ends;  // the accumulators are never free this early
          if (!run_ends && j == 0) ok = mbar_test(a_ready + 8 * (g1 & 3), (g1 >> 2) & 1);
          if (elected) small_products(tmem_u + 128, ta, wb, 0, 3, c % EX_RUN == 0);
          __syncwarp();
          ok = mbar_test(w_ready + 8 * slot1, phase1 & 1) && ok;
          if (elected) small_products(tmem_u + 128, ta, wb, 3, 4, false);
          __syncwarp();
          if (elected) {
            if (j == per_item - 1) mma_commit(a_done + 8 * ab);
            mma_commit(w_done + 8 * slot);
            if (run_ends) mma_commit(d_full);
          }
          if (run_ends) ++run;
          open = __all_sync(0xffffffffu, ok);
          slot = slot1;
          phase = phase1;
        }
      }
      g += nch;
    }
    drain_mma(retired, elected);
  } else if (warp == PS_TMA_WARP) {
    uint32_t elected;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(elected));
    const uint32_t ring_u = __shfl_sync(0xffffffffu, ring, 0);
    bool alive = true;
    uint32_t wu = 0, slot = 0, phase = 0;
    for (int item = blockIdx.x; alive && walk.seek(item / per_tile, e, s0, rows); item += gridDim.x) {
      for (int j = 0; j < per_item && alive; ++j) {
        const int row = e * d.n_out + 128 * (shared ? j : item % nb);
        for (int c = 0; c < nch; ++c, ++wu) {
          if (phase > 0) alive = mbar_wait(w_done + 8 * slot, (phase - 1) & 1);
          alive = __all_sync(0xffffffffu, alive);
          if (!alive) break;
          if (elected) {
            const uint32_t bar = w_ready + 8 * slot, dst = ring_u + slot * 2 * TC_TILE_BYTES;
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(2 * TC_TILE_BYTES) : "memory");
            tma_load_2d(dst, &maps.hi, bar, c * TC_BK, row);
            tma_load_2d(dst + TC_TILE_BYTES, &maps.lo, bar, c * TC_BK, row);
          }
          __syncwarp();
          if (++slot == EX_W_SLOTS) { slot = 0; ++phase; }
        }
      }
    }
    drain_copies(w_ready, EX_W_SLOTS, wu);
  } else if (warp >= EX_EPI_WARP0) {
    // thread = row; epilogue warp e takes columns 64 (e >> 2).. of the accumulator
    const int quarter = warp & 3, half = (warp - EX_EPI_WARP0) >> 2;
    const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * 64);
    const bool wide = ((reinterpret_cast<uintptr_t>(d.y) | reinterpret_cast<uintptr_t>(d.gate)) & 31u) == 0 && d.ld_y % 8 == 0 && d.ld_gate % 8 == 0;
    float* const bias = reinterpret_cast<float*>(smem + EX_BIAS_OFF) + 64 * (warp - EX_EPI_WARP0);
    *reinterpret_cast<float2*>(bias + 2 * lane) = make_float2(0.f, 0.f);
    bool alive = true;
    uint32_t run = 0;
    for (int item = blockIdx.x; walk.seek(item / per_tile, e, s0, rows); item += gridDim.x) {
      for (int jj = 0; jj < per_item; ++jj) {
        const int c0 = 128 * (shared ? jj : item % nb) + 64 * half;
        const bool valid = quarter * 32 + lane < rows;
        const int64_t slot = s0 + (valid ? quarter * 32 + lane : 0);
        const float* const gate = d.gate ? d.gate + slot * d.ld_gate + c0 : nullptr;
        float* const out = d.y + slot * d.ld_y + c0;
        // the products wait for the accumulators: no load from memory may stand between their reads
        __syncwarp();
        if (d.bias) *reinterpret_cast<float2*>(bias + 2 * lane) = *reinterpret_cast<const float2*>(d.bias + (int64_t)e * d.n_out + c0 + 2 * lane);
        __syncwarp();
        if (gate) {
          asm volatile("prefetch.global.L2 [%0];" :: "l"(gate));
          asm volatile("prefetch.global.L2 [%0];" :: "l"(gate + 32));
        }
        for (int c_run = 0; c_run < nch; c_run += EX_RUN, ++run) {
          const bool first = c_run == 0, last = c_run + EX_RUN >= nch;
          if (alive) alive = mbar_wait(d_full, run & 1);
          alive = __all_sync(0xffffffffu, alive);
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
          for (int cg = 0; cg < 4; ++cg) {
            uint32_t v[16], u[16];
            __syncwarp();  // lanes without a row have skipped the previous columns' work; these reads want the whole warp
            MB_TMEM_LD16(lane_base + 16u * cg, v);
            MB_TMEM_LD16(lane_base + 128u + 16u * cg, u);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            if (cg == 3) {
              asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
              __syncwarp();
              if (lane == 0) mbar_arrive(d_free);
            }
            if (!alive || !valid) continue;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int c = cg * 16 + q * 8;
              float o[8];
#pragma unroll
              for (int i = 0; i < 8; i += 2)
                apart(two(__uint_as_float(v[8 * q + i]), __uint_as_float(v[8 * q + i + 1])) +
                          two(__uint_as_float(u[8 * q + i]), __uint_as_float(u[8 * q + i + 1])),
                      o[i], o[i + 1]);
              if (!first) {  // what this thread left there
                add4_to(o, ld4(out + c));
                add4_to(o + 4, ld4(out + c + 4));
              }
              if (last) {
                add4_to(o, ld4(bias + c));
                add4_to(o + 4, ld4(bias + c + 4));
                if (gate) {
                  silu_grad4_to(o, ld4(gate + c));
                  silu_grad4_to(o + 4, ld4(gate + c + 4));
                }
                if (d.out_act) silu_fast_all(o, o);
              }
              if (wide) st8(out + c, o);
              else { st4(out + c, make_float4(o[0], o[1], o[2], o[3])); st4(out + c + 4, make_float4(o[4], o[5], o[6], o[7])); }
            }
          }
        }
      }
    }
  } else {
    // producers: lane quarter, every fourth K chunk; thread = row = TMEM lane
    const int pw = warp - PS_PROD_WARP0, set = pw >> 2, quarter = warp & 3, lr = lane >> 3, lc = lane & 7;
    const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const uint32_t patch0 = smem_u32(smem + EX_PATCH_OFF + pw * (EX_STAGES * 32 * 128));
    const uint32_t put_even = lr * 128 + ((lc ^ lr) << 4), put_odd = lr * 128 + ((lc ^ (lr | 4)) << 4);
    // The walk is that of the chunks asked for, EX_STAGES - 1 ahead of those converted; the rows of an item are looked up a chunk before
    // they are needed.  This warp's n-th chunk is chunk 4 n + set of the CTA
    // and goes to A buffer `set`.
    int item = blockIdx.x, g_c = 0, asked = 0;
    int32_t a_row[8], next_row[8];
    bool more;
    const float* const x = d.x + set * TC_BK + 4 * lc;
    auto look_up = [&]() {
      more = walk.seek(item / per_tile, e, s0, rows);
      if (!more) return;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = quarter * 32 + lr + 4 * i;
        const int64_t s = s0 + (r < rows ? r : rows - 1);
        next_row[i] = d.idx ? d.idx[s] : (int32_t)s;
      }
    };
    auto request = [&]() {     // this warp's next chunk into its next patch
      if (more) {
        if (g_c == 0) {
#pragma unroll
          for (int i = 0; i < 8; ++i) a_row[i] = (int32_t)min(max((int64_t)next_row[i], (int64_t)0), d.n_rows - 1);
        }
        const uint32_t to = patch0 + (uint32_t)(asked % EX_STAGES) * (32 * 128);
        const float* const from = x + EX_SETS * TC_BK * g_c;
#pragma unroll
        for (int i = 0; i < 8; ++i) copy16(to + ((i & 1) ? put_odd : put_even) + 512u * i, from + (int64_t)a_row[i] * (int)d.ld_x);
        ++asked;
        if (++g_c == nch / EX_SETS) { g_c = 0; item += gridDim.x; look_up(); }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    look_up();
    for (int i = 0; i < EX_STAGES - 1; ++i) request();
    bool alive = true;
    for (int n = 0; ; ++n) {
      request();  // into the patch read one chunk ago; the __syncwarp that closed that chunk orders the reads
      if (n >= asked) break;
      asm volatile("cp.async.wait_group %0;" :: "n"(EX_STAGES - 1) : "memory");
      __syncwarp();
      const uint32_t patch = patch0 + (uint32_t)(n % EX_STAGES) * (32 * 128), ta = lane_base + 256 + 64 * set;
      auto values = [&](int h, float (&v)[8]) {  // a quarter of this row's 32
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float4 f = lds4(patch + lane * 128 + (((2 * h + i) ^ (lane & 7)) << 4));
          v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
        }
        if (d.in_act) silu_fast_all(v, v);
      };
      f2 seen = two(0.f, 0.f);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        float v[8];
        values(h, v);
        uint32_t hi[8], lo[8];
        split_tf32_all(v, hi, lo, seen);
        if (h == 0) {
          if (n > 0 && alive) alive = mbar_wait(a_done + 8 * set, (n - 1) & 1);  // the A buffer is free again
          alive = __all_sync(0xffffffffu, alive);
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        }
        MB_TMEM_ST8(ta + 8 * h, hi);
        MB_TMEM_ST8(ta + 32 + 8 * h, lo);
      }
      if (split_again(seen)) {
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");  // the parts above are written over
#pragma unroll 1
        for (int h = 0; h < 4; ++h) {
          float v[8];
          values(h, v);
          uint32_t hi[8], lo[8];
          split_tf32_large(v, hi, lo);
          __syncwarp();
          MB_TMEM_ST8(ta + 8 * h, hi);
          MB_TMEM_ST8(ta + 32 + 8 * h, lo);
        }
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(a_ready + 8 * set);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  }

  if (d.zero_rest) {  // slots ahead of the first expert's and behind the last one's
    const int64_t first = min(max((int64_t)d.offsets[0], (int64_t)0), d.n_slots);
    const int64_t used = min(max((int64_t)d.offsets[d.n_experts], first), d.n_slots), skip = used - first;
    for (int64_t i = (int64_t)blockIdx.x * (EX_THREADS / 32) + warp; i < d.n_slots - skip; i += (int64_t)gridDim.x * (EX_THREADS / 32)) {
      const int64_t s = i < first ? i : i + skip;
      for (int c = 4 * lane; c < d.n_out; c += 128) st4(d.y + s * d.ld_y + c, make_float4(0.f, 0.f, 0.f, 0.f));
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == PS_MMA_WARP) {
    __syncwarp();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem_base), "r"(PS_TMEM_COLS) : "memory");
  }
}

// w [n_out, n_in] of every expert -> tf32 parts hi, lo, and both transposed; 32 x 32 values a block
__global__ void __launch_bounds__(256) k_experts_split(int n_out, int n_in, int64_t part, const float* __restrict__ w, float* __restrict__ parts) {
  pdl_sync();
  __shared__ float t[2][32][33];
  const int64_t e0 = (int64_t)blockIdx.z * n_out * n_in;
  const int k0 = blockIdx.x * 32, n0 = blockIdx.y * 32, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
#pragma unroll
  for (int i = ty; i < 32; i += 8) {
    const int64_t at = e0 + (int64_t)(n0 + i) * n_in + k0 + tx;
    const float x = w[at];
    float hi = to_tf32(x), lo = to_tf32(x - hi);
    if (!(fabsf(hi) <= FLT_MAX)) {  // as in split_tf32_large
      hi = fabsf(x) <= FLT_MAX ? __uint_as_float(__float_as_uint(x) & 0xFFFFE000u) : 0.f;
      lo = to_tf32(x - hi);
    }
    parts[at] = hi;
    parts[part + at] = lo;
    t[0][i][tx] = hi;
    t[1][i][tx] = lo;
  }
  __syncthreads();
#pragma unroll
  for (int i = ty; i < 32; i += 8) {
    const int64_t at = e0 + (int64_t)(k0 + i) * n_out + n0 + tx;
    parts[2 * part + at] = t[0][tx][i];
    parts[3 * part + at] = t[1][tx][i];
  }
}

// ------------------------------------------------------------------ weight gradient
// dW_e = sum over the slots of e of dy[s]^T f(x[idx[s]]): the contraction runs over rows, so both operands have to be turned.  A
// thread that holds a COLUMN does that for free: lanes of a warp read 32 neighbouring values of a row, row after row, and own one
// column each.  dy columns (lane = row of dW) go to tensor memory as the A operand, x columns to shared memory as the K-major B
// operand, in chunks of 32 rows, both as two tf32 parts (k_experts has the arithmetic).
//
// Work is cut by rows, not by experts: the chunks of all experts, numbered through, are shared out evenly over the CTAs of a 128 x 128
// block of dW (a share may begin and end inside an expert), so that one expert with most rows costs no more than even ones.  A run of
// chunks that holds all of an expert goes straight to dW; the others, two a share at the most, are left as partial sums and joined in
// order by k_experts_grad_join.
//
// The tensor cores cut each sum they accumulate to float32 instead of rounding it, always towards zero: after n of them a sum is
// short by up to n 2^-23.  So a run is accumulated there for EG_FLUSH chunks only and added up in float32 registers of the epilogue
// warps, rounded to nearest; after EG_FOLD such sums, 4,096 rows, these go to their place in memory and start again, so that no chain of
// additions grows with the number of rows but that of the 4,096s (the bias gradient's are added in 64 bits).
//
// 573,894 slots, 256 -> 128, 32 experts: 315 us (119 TFLOP/s).  The column warps bound it, some 2,000 cycles a chunk of their own
// instructions where its products take 768; sixteen of them do not fit the registers beside the epilogue's sums.
//
// Roles: warp 0 issues the products, warps 2 - 5 hold dy's columns, 6 - 9 x's, 10 - 17 the sums (warp 1 has none).
constexpr int EG_FLUSH = 4, EG_FOLD = 32;
constexpr int EG_BUFS = 4;
constexpr int EG_STAGES = 3;
constexpr int EG_PATCH_OFF = EG_BUFS * 2 * TC_TILE_BYTES;
constexpr int EG_BAR_OFF = EG_PATCH_OFF + 8 * EG_STAGES * 32 * 128;
constexpr int EG_SMEM_BYTES = EG_BAR_OFF + 256;
static_assert(EG_SMEM_BYTES <= 227 * 1024, "shared memory of one CTA");

struct GradShare {  // chunks [lo, hi) of share c of n
  int64_t all, lo, hi;
  __device__ __forceinline__ GradShare(int64_t all_, int c, int n) : all(all_), lo(all_ * c / n), hi(all_ * (c + 1) / n) {}
  static __device__ __forceinline__ int of(int64_t chunk, int64_t all, int n) { return (int)(((chunk + 1) * n - 1) / all); }
};

__global__ void __launch_bounds__(PS_THREADS, 1)
k_experts_grad(const __grid_constant__ mb_experts d, const int n_share, float* const part, float* const part_bias) {
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + EG_BAR_OFF);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + EG_BAR_OFF + 240);
  // of an accumulator: -3: the run goes on; otherwise the run's sum goes to place (what >> 1) - 2, added to what it has left there before, and
  // ends with what & 1.  Place -2 / -1: the share's first / second partial sum, e >= 0: all of expert e.  -4: the share is done
  volatile int32_t* const target = reinterpret_cast<volatile int32_t*>(smem + EG_BAR_OFF + 224);
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) atomicOr(&g_gemm_status, 2);
    return;
  }
  // ready[4] (8 column warps) done[4] | d_full[2] d_free[2] (8 epilogue warps) | retired | told[2] (where a finished accumulator goes)
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t ready = bar0, done = bar0 + 32, d_full = bar0 + 64, d_free = bar0 + 80, retired = bar0 + 96, told = bar0 + 104;
  const uint32_t tiles = smem_u32(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nk = d.n_in / 128, nb = nk * (d.n_out / 128);
  const int c = blockIdx.x / nb, n0 = 128 * (blockIdx.x % nb / nk), k0 = 128 * (blockIdx.x % nk);

  if (warp == PS_MMA_WARP) {
    if (lane == 0) {
      for (int b = 0; b < 4; ++b) { mbar_init(ready + 8 * b, 8); mbar_init(done + 8 * b, 1); }
      for (int b = 0; b < 2; ++b) { mbar_init(d_full + 8 * b, 1); mbar_init(d_free + 8 * b, 8); mbar_init(told + 8 * b, 1); }
      mbar_init(retired, 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 :: "r"(smem_u32(tmem_slot)), "r"(PS_TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = *tmem_slot;
  pdl_sync();
  Walk<5> walk;
  walk.start(d);
  const GradShare share(walk.count(), c, n_share);
  int e;
  int64_t s0, left;
  bool first;
  bool alive = true;

  if (warp == PS_MMA_WARP) {
    uint32_t elected;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(elected));
    const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem_base, 0), tiles_u = __shfl_sync(0xffffffffu, tiles, 0);
    uint32_t g = 0, k = 0, in_acc = 0, sums = 0;  // sums of the run in the epilogue's registers
    bool fresh = true, from_start = false;
    auto tell = [&](int32_t what) {
      if (lane == 0) {
        target[k & 1] = what;
        mbar_arrive(told + 8 * (k & 1));
      }
    };
    left = 0;
    for (int64_t t = share.lo; t < share.hi && walk.next((int)t, e, s0, left, first); ++t, ++g) {
      const uint32_t b = g & 3, acc = k & 1;
      if (fresh) { from_start = first; fresh = false; }
      if (in_acc == 0 && k >= 2 && alive) alive = mbar_wait(d_free + 8 * acc, ((k >> 1) - 1) & 1);
      if (alive) alive = mbar_wait(ready + 8 * b, (g >> 2) & 1);
      alive = __all_sync(0xffffffffu, alive);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const bool end = left <= 32 || t + 1 == share.hi;
      const bool flush = in_acc == EG_FLUSH - 1 || end;
      if (flush) {
        ++sums;
        if (end || sums == EG_FOLD) {
          const bool all = from_start && left <= 32 * (share.hi - t);  // the expert ends in this share too
          tell(2 * ((all ? e : from_start ? -1 : -2) + 2) + (end ? 1 : 0));
          sums = 0;
        } else {
          tell(-3);
        }
      }
      // from one lane, so that the operands of the matrix instructions are the same for all by construction (see k_experts)
      const uint32_t how = __shfl_sync(0xffffffffu, b | acc << 2 | (in_acc == 0 ? 8u : 0u) | (flush ? 16u : 0u), 0);
      const uint32_t ub = how & 3, uacc = how >> 2 & 1;
      if (elected) {
        issue_chunk_mmas<false>(tmem_u + 128u * uacc, tmem_u + 256 + 64 * ub, tiles_u + ub * 2 * TC_TILE_BYTES, 0, (how & 8) != 0);
        mma_commit(done + 8 * ub);
        if (how & 16) mma_commit(d_full + 8 * uacc);
      }
      __syncwarp();
      ++in_acc;
      if (flush) { in_acc = 0; ++k; }
      if (end) fresh = true;
    }
    if (k >= 2 && alive) alive = mbar_wait(d_free + 8 * (k & 1), ((k >> 1) - 1) & 1);
    tell(-4);
    drain_mma(retired, elected);
  } else if (warp >= PS_EPI_WARP0) {
    // thread = row of the block, 64 of its columns; sums of a run in registers
    const int quarter = warp & 3, half = (warp - PS_EPI_WARP0) >> 2;
    const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * 64);
    const int64_t at = (int64_t)(n0 + quarter * 32 + lane) * d.n_in + k0 + 64 * half, whole = (int64_t)d.n_out * d.n_in;
    f2 sum[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) sum[i] = two(0.f, 0.f);
    bool more = false;  // this run has left a sum at its place before
    for (uint32_t k = 0; ; ++k) {
      const uint32_t acc = k & 1;
      if (alive) alive = mbar_wait(told + 8 * acc, (k >> 1) & 1);
      alive = __all_sync(0xffffffffu, alive);
      const int what = alive ? target[acc] : -4;
      if (what == -4) break;
      if (alive) alive = mbar_wait(d_full + 8 * acc, (k >> 1) & 1);
      alive = __all_sync(0xffffffffu, alive);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
      for (int cg = 0; cg < 4; ++cg) {
        uint32_t v[16];
        MB_TMEM_LD16(lane_base + 128u * acc + 16u * cg, v);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[8 * cg + i] = sum[8 * cg + i] + two(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(d_free + 8 * acc);
      if (what == -3) continue;
      const int place = (what >> 1) - 2;
      float* const out = (place >= 0 ? d.dw + place * whole : part + (2 * c + 2 + place) * whole) + at;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float o[4];
        apart(sum[2 * i], o[0], o[1]);
        apart(sum[2 * i + 1], o[2], o[3]);
        if (more) add4_to(o, ld4(out + 4 * i));
        if (alive) st4(out + 4 * i, make_float4(o[0], o[1], o[2], o[3]));
        sum[2 * i] = sum[2 * i + 1] = two(0.f, 0.f);
      }
      more = !(what & 1);
    }
  } else if (warp >= PS_PROD_WARP0) {
    // columns: warps 2 - 5 dy (A, tensor memory), 6 - 9 x (B, shared memory), 32 columns each
    const bool is_x = warp >= PS_PROD_WARP0 + 4;
    const int quarter = warp & 3, col = 32 * quarter + lane;
    const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16) + 256;
    // A chunk's 32 rows x 32 columns come by cp.async into a patch of the warp's own, EG_STAGES - 1 chunks ahead, and are read back by
    // column: 32 lanes, 32 neighbouring words.  (With plain loads into registers a chunk ahead the warps waited for the loads just
    // issued: 717 us where this takes 300.)
    const int lr = lane >> 3, lc = lane & 7;
    const uint32_t patch0 = tiles + EG_PATCH_OFF + (warp - PS_PROD_WARP0) * (EG_STAGES * 32 * 128);
    int row = 0, asked = 0;    // lane's row of the next chunk to ask for (x: in the source), looked up a chunk earlier
    int rows = 0;
    int64_t t_next = share.lo;
    const float* const base = (is_x ? d.x + k0 : d.dy + n0) + 32 * quarter + 4 * lc;
    const int ld = (int)(is_x ? d.ld_x : d.ld_dy);
    left = 0;
    auto look_up = [&]() {
      rows = 0;
      if (t_next < share.hi && walk.next((int)t_next, e, s0, left, first)) {
        rows = left < 32 ? (int)left : 32;
        row = lane < rows ? (is_x && d.idx ? d.idx[s0 + lane] : (int32_t)(s0 + lane)) : 0;
      }
      ++t_next;
    };
    auto request = [&]() {
      if (rows > 0) {
        const int r = is_x ? (int)min(max((int64_t)row, (int64_t)0), d.n_rows - 1) : row;
        const uint32_t to = patch0 + (uint32_t)(asked % EG_STAGES) * (32 * 128) + lr * 128 + lc * 16;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float* const from = base + (int64_t)__shfl_sync(0xffffffffu, r, lr + 4 * i) * ld;
          const int bytes = lr + 4 * i < rows ? 16 : 0;  // 0: nothing is read, zeros are written
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(to + 512u * i), "l"(from), "r"(bytes) : "memory");
        }
        ++asked;
        look_up();
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    look_up();
    for (int i = 0; i < EG_STAGES - 1; ++i) request();
    // what the bias gradient needs, chunk by chunk, from a walk of its own
    Walk<5> now = walk;
    int e0 = 0;
    int64_t now_s = 0, now_left = 0;
    bool first0 = false;
    if (!is_x) { now.start(d); }
    uint32_t g = 0;
    float bias = 0.f;
    double bias_sum = 0.;
    int summed = 0;  // chunks in `bias`
    bool fresh = true, from_start = false;
    for (int64_t t = share.lo; t < share.hi; ++t, ++g) {
      const uint32_t b = g & 3;
      request();  // into the patch read one chunk ago; the __syncwarp that closed that chunk orders the reads
      asm volatile("cp.async.wait_group %0;" :: "n"(EG_STAGES - 1) : "memory");
      __syncwarp();
      const uint32_t patch = patch0 + (g % EG_STAGES) * (32 * 128) + lane * 4;
      if (g >= 4 && alive) alive = mbar_wait(done + 8 * b, ((g >> 2) - 1) & 1);
      alive = __all_sync(0xffffffffu, alive);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t line = tiles + b * 2 * TC_TILE_BYTES + col * 128;
      auto values = [&](int h, float (&x)[8]) {  // a quarter of this column's 32
#pragma unroll
        for (int i = 0; i < 8; ++i) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x[i]) : "r"(patch + 128u * (8 * h + i)) : "memory");
        if (is_x && d.in_act) silu_fast_all(x, x);
      };
      auto put = [&](int h, const uint32_t (&hi)[8], const uint32_t (&lo)[8]) {
        if (is_x) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t to = line + (((2 * h + i) ^ (col & 7)) << 4);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                         :: "r"(to), "r"(hi[4 * i]), "r"(hi[4 * i + 1]), "r"(hi[4 * i + 2]), "r"(hi[4 * i + 3]) : "memory");
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                         :: "r"(to + TC_TILE_BYTES), "r"(lo[4 * i]), "r"(lo[4 * i + 1]), "r"(lo[4 * i + 2]), "r"(lo[4 * i + 3]) : "memory");
          }
        } else {
          MB_TMEM_ST8(lane_base + 64 * b + 8 * h, hi);
          MB_TMEM_ST8(lane_base + 64 * b + 32 + 8 * h, lo);
        }
      };
      f2 seen = two(0.f, 0.f);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        uint32_t hi[8], lo[8];
        float x[8];
        values(h, x);
        if (!is_x) bias += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        split_tf32_all(x, hi, lo, seen);
        put(h, hi, lo);
      }
      if (split_again(seen)) {
        if (!is_x) asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");  // the parts above are written over
#pragma unroll 1
        for (int h = 0; h < 4; ++h) {
          uint32_t hi[8], lo[8];
          float x[8];
          values(h, x);
          split_tf32_large(x, hi, lo);
          __syncwarp();
          put(h, hi, lo);
        }
      }
      if (is_x) {
        to_async_proxy();
      } else {
        now.next((int)t, e0, now_s, now_left, first0);
        const bool last0 = now_left <= 32;
        if (fresh) { from_start = first0; fresh = false; }
        const bool end = last0 || t + 1 == share.hi;
        if (++summed == EG_FOLD * EG_FLUSH || end) {
          bias_sum += (double)bias;
          bias = 0.f;
          summed = 0;
        }
        if (end) {
          if (part_bias && k0 == 0) {
            float* const out = from_start && last0 ? d.dbias + (int64_t)e0 * d.n_out : part_bias + (int64_t)(2 * c + (from_start ? 1 : 0)) * d.n_out;
            out[n0 + col] = (float)bias_sum;
          }
          bias_sum = 0.;
          fresh = true;
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(ready + 8 * b);
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == PS_MMA_WARP) {
    __syncwarp();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem_base), "r"(PS_TMEM_COLS) : "memory");
  }
}

// The partial sums of experts whose slots lie in more than one share, in order of share; zeros for experts without slots.
// blockIdx.y = expert; the bias gradient is the last n_out values of an expert's part
__global__ void __launch_bounds__(256) k_experts_grad_join(const __grid_constant__ mb_experts d, const int n_share, const float* __restrict__ part,
                                                           const float* __restrict__ part_bias) {
  pdl_sync();
  const int e = blockIdx.y;
  Walk<5> walk;
  walk.start(d);
  int64_t before = 0, mine = 0, all = 0;
  for (int b = 0; b < d.n_experts; b += 32) {
    walk.base = b;
    walk.load();
    if (e >= b && e < b + 32) {
      const int upto = __shfl_sync(0xffffffffu, walk.upto, e - b), ahead = __shfl_sync(0xffffffffu, walk.upto, e > b ? e - b - 1 : 0);
      before = all + (e > b ? ahead : 0);
      mine = all + upto - before;
    }
    all += walk.total;
  }
  int c0 = 0, c1 = 0;
  if (mine > 0) {
    c0 = GradShare::of(before, all, n_share);
    c1 = GradShare::of(before + mine - 1, all, n_share);
    if (c0 == c1) return;  // in dW already
  }
  const int64_t whole = (int64_t)d.n_out * d.n_in;
  const int64_t i = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x);
  const bool is_bias = i >= whole;
  if (is_bias && (!d.dbias || i >= whole + d.n_out)) return;
  const int64_t stride = is_bias ? d.n_out : whole, at = is_bias ? i - whole : i;
  const float* const from = is_bias ? part_bias : part;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (mine > 0) {
    s = ld4(from + (2 * (int64_t)c0 + 1) * stride + at);
    for (int c = c0 + 1; c <= c1; ++c) {
      const GradShare share(all, c, n_share);
      if (share.lo < share.hi) s = add4(s, ld4(from + 2 * (int64_t)c * stride + at));
    }
  }
  st4((is_bias ? d.dbias : d.dw) + e * stride + at, s);
}
