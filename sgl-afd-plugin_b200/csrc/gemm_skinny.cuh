// FP8 block-scaled linear for few rows: the weight tile is the MMA's 128-row operand, the rows of x its columns, and the
// K blocks of a tile are split over a cluster of S CTAs.  Included by linear.cu.
//
// With few rows the cost is reading the weights once, and the launches.  Splitting K makes 100 to 300 CTAs of a product
// that has 16 to 56 weight tiles, so that most of the weights are in flight at once; the cluster adds its S partial
// tiles through distributed shared memory in rank order: no partial sums in memory, no second kernel, the same bits every
// time.  A handful of rows is quantised by every CTA for its own K blocks (a few KB, from L2) while TMA already fetches the
// weights, and the product is one launch.  With more rows the repeated quantisation costs more than a launch: the rows
// come quantised (XTMA), by TMA beside the weights, from a kernel that this one overlaps: it is launched programmatically,
// and its weights do not wait for that kernel.
#pragma once

namespace lin {

constexpr int SK_FOLD_WARPS = 8, SK_THREADS = 32 * (2 + SK_FOLD_WARPS);
constexpr int SK_MAX_KB = 64, SK_MAX_STAGES = 12, SK_MAX_SPLIT = 8;

template <int TN, int SWIGLU, int XTMA>
struct Skinny {
  static constexpr int TILES = SWIGLU ? 2 : 1;          // weight tiles of 128 rows per CTA (gate and up)
  static constexpr int W_BYTES = TILES * 128 * BK;
  static constexpr int STAGE_BYTES = W_BYTES + (XTMA ? TN * BK : 0);
  static constexpr int ACC_COLS = TILES * TN;           // TMEM columns of one K block's partial
  static constexpr int C = ACC_COLS / 2;                // columns per folding warp
  static constexpr int TMEM = C <= 32 ? 256 : 512;      // columns of tensor memory: two CTAs on an SM, or one
  static constexpr int BUFS = TMEM / ACC_COLS;
  static constexpr int G = C == 64 ? 32 : C == 32 ? 16 : C;  // columns per TMEM load
  static_assert(BUFS >= 2, "two partials at least");
};

struct SkinnyParams {
  CUtensorMap tmap_w;  // weights [N, K]
  CUtensorMap tmap_x;  // XTMA: codes [M, 128 KB], boxes of tn rows
  const uint16_t* x;
  int64_t ldx;
  int32_t M, K, N, KB, NB, split, stages, max_kb, tn;
  const float* sb;
  int32_t fp16, pow2;
  void* out;  // linear: [M, N] of x's type
  float swiglu_limit;
  uint8_t* out_q;  // SwiGLU: codes of h [M, N / 2]
  float* out_sa;   // SwiGLU: scales of h [N / 256][mp]
  int64_t mp;
  const float* sa;  // XTMA: scales [KB][mp]
  uint64_t status, timeout_ns;
};

// Programmatic launch: wait until the kernels this one was launched beside have finished, and let the next one start.
__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dependents_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ float4 peer_load4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}
// The sum of the cluster's words at one shared-memory address, in rank order, all loads in flight before the first add
__device__ __forceinline__ float4 cluster_sum(uint32_t addr, int S) {
  float4 v[SK_MAX_SPLIT];
#pragma unroll
  for (int s = 0; s < SK_MAX_SPLIT; ++s)
    if (s < S) v[s] = peer_load4(peer_addr(addr, s));
  float4 a = v[0];
#pragma unroll
  for (int s = 1; s < SK_MAX_SPLIT; ++s)
    if (s < S) a.x += v[s].x, a.y += v[s].y, a.z += v[s].z, a.w += v[s].w;
  return a;
}
__device__ __forceinline__ void tmem_ld_32x32b_x8(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

template <int G>
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&v)[G]) {
  if constexpr (G == 8) tmem_ld_32x32b_x8(taddr, v);
  else if constexpr (G == 16) tmem_ld_32x32b_x16(taddr, v);
  else tmem_ld_32x32b_x32(taddr, v);
}
// tcgen05.wait::ld that the uses of `v` cannot be moved above
template <int G>
__device__ __forceinline__ void tmem_wait_cols(uint32_t (&v)[G]) {
  if constexpr (G == 32) {
    tmem_wait_regs(v);
  } else if constexpr (G == 16) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                   "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]),
                   "+r"(v[15])
                 :
                 : "memory");
  } else {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7])
                 :
                 : "memory");
  }
}
// acc[c] += v[c] * (sa[c] * sb)
template <int G>
__device__ __forceinline__ void fold_cols(float* acc, const uint32_t (&v)[G], const float* sa, float sb) {
#pragma unroll
  for (int c = 0; c < G; c += 4) {
    const float4 f = *reinterpret_cast<const float4*>(sa + c);
    acc[c] = fmaf(__uint_as_float(v[c]), f.x * sb, acc[c]);
    acc[c + 1] = fmaf(__uint_as_float(v[c + 1]), f.y * sb, acc[c + 1]);
    acc[c + 2] = fmaf(__uint_as_float(v[c + 2]), f.z * sb, acc[c + 2]);
    acc[c + 3] = fmaf(__uint_as_float(v[c + 3]), f.w * sb, acc[c + 3]);
  }
}

template <int TN, int SWIGLU, int XTMA>
__global__ void __launch_bounds__(SK_THREADS, Skinny<TN, SWIGLU, XTMA>::C <= 32 ? 2 : 1)
    linear_skinny_kernel(const __grid_constant__ SkinnyParams p) {
  using T = Skinny<TN, SWIGLU, XTMA>;
  constexpr int C = T::C;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sW = smem;                            // [stages][TILES][128 rows x 128 B], XTMA: [TN rows x 128 B]
  uint8_t* sX = sW + p.stages * T::STAGE_BYTES;  // not XTMA: [max_kb][TN rows x 128 B]
  float* sSa = reinterpret_cast<float*>(sX + (XTMA ? 0 : p.max_kb * TN * BK));  // [max_kb][TN]
  float* sSb = sSa + p.max_kb * TN;                     // [max_kb][2]
  uint64_t* full = reinterpret_cast<uint64_t*>(sSb + 2 * p.max_kb);
  uint64_t* empty = full + SK_MAX_STAGES;
  uint64_t* x_full = empty + SK_MAX_STAGES;  // not XTMA: every folding warp has written its part of x
  uint64_t* acc_full = x_full + 1;           // [BUFS <= 16]
  uint64_t* acc_empty = acc_full + 16;
  uint64_t* mma_done = acc_empty + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank(), S = p.split;
  const int n_t = blockIdx.x / S;
  const int row0 = blockIdx.y * p.tn, rows = min(p.tn, p.M - row0);
  const int kb0 = rank * p.KB / S, kbs = (rank + 1) * p.KB / S - kb0;
  {  // one thread per barrier: initialised by one thread they take longer than the first weights
    const int t = threadIdx.x;
    if (t < p.stages) {
      mbar_init(&full[t], 1);
      mbar_init(&empty[t], 1);
    }
    if (t < T::BUFS) {
      mbar_init(&acc_full[t], 1);
      mbar_init(&acc_empty[t], SK_FOLD_WARPS);
    }
    if (t == 32) {
      mbar_init(x_full, SK_FOLD_WARPS);
      mbar_init(mma_done, 1);
      *abort_flag = 0;
    }
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, T::TMEM);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) prefetch_tmap(&p.tmap_w);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint64_t deadline = globaltimer_ns() + p.timeout_ns;
  bool ok = true;

  if (warp == 0) {
    if (lane == 0) {
      const int b0 = n_t * 128, b1 = p.N / 2 + n_t * 128;
      const uint32_t tx = T::W_BYTES + (XTMA ? p.tn * BK : 0);
      auto weights = [&](int i, int stage) {
        uint8_t* dst = sW + stage * T::STAGE_BYTES;
        mbar_arrive_expect_tx(&full[stage], tx);
        tma_load_2d(dst, &p.tmap_w, (kb0 + i) * BK, b0, &full[stage]);
        if constexpr (SWIGLU) tma_load_2d(dst + 128 * BK, &p.tmap_w, (kb0 + i) * BK, b1, &full[stage]);
      };
      // the weights depend on no other kernel
      const int first = min(kbs, p.stages);
      for (int i = 0; i < first; ++i) weights(i, i);
      if constexpr (XTMA) grid_dependency_wait();
      int stage = 0;
      uint32_t phase = 0;
      for (int i = 0; i < kbs; ++i) {
        if (i >= first) {
          ok = mbar_wait(&empty[stage], phase ^ 1u, deadline, abort_flag);
          if (!ok) break;
          weights(i, stage);
        }
        if constexpr (XTMA)
          tma_load_2d(sW + stage * T::STAGE_BYTES + T::W_BYTES, &p.tmap_x, (kb0 + i) * BK, row0, &full[stage]);
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    const uint32_t idesc = idesc_f8f6f4(128, p.tn);
    int stage = 0;
    uint32_t phase = 0;
    if (!XTMA) ok = __all_sync(0xffffffffu, mbar_wait(x_full, 0, deadline, abort_flag));
    for (int i = 0; ok && i < kbs; ++i) {
      const uint32_t buf = i % T::BUFS;
      const uint8_t* w = sW + stage * T::STAGE_BYTES;
      const uint64_t wdesc = sdesc_sw128(w), xdesc = sdesc_sw128(XTMA ? w + T::W_BYTES : sX + i * TN * BK);
      ok = (i < T::BUFS || mbar_wait(&acc_empty[buf], ((i / T::BUFS) & 1u) ^ 1u, deadline, abort_flag)) &&
           mbar_wait(&full[stage], phase, deadline, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int h = 0; h < T::TILES; ++h)
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            tc_mma_f8f6f4(tmem_base + buf * T::ACC_COLS + h * TN, wdesc + (uint64_t)(h * 128 * BK >> 4) + 2ull * k,
                          xdesc + 2ull * k, idesc, k != 0);
        tc_commit(&acc_full[buf]);
        if (i + p.stages < kbs) tc_commit(&empty[stage]);
      }
      __syncwarp();
      if (++stage == p.stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (elect_one()) tc_commit(mma_done);
    __syncwarp();
    drain_mmas(mma_done, deadline, abort_flag);
  } else {
    const int fw = warp - 2, ft = threadIdx.x - 64;
    for (int i = ft; i < kbs; i += 32 * SK_FOLD_WARPS) {
      sSb[2 * i] = __ldg(p.sb + (int64_t)n_t * p.KB + kb0 + i);
      sSb[2 * i + 1] = SWIGLU ? __ldg(p.sb + (int64_t)(p.NB / 2 + n_t) * p.KB + kb0 + i) : 0.f;
    }
    if constexpr (XTMA) {
      grid_dependency_wait();
      for (int i = ft; i < kbs * TN; i += 32 * SK_FOLD_WARPS) {
        const int kb = i / TN, r = i % TN;
        sSa[i] = r < rows ? p.sa[(int64_t)(kb0 + kb) * p.mp + row0 + r] : 0.f;
      }
      asm volatile("bar.sync 1, %0;" ::"n"(32 * SK_FOLD_WARPS) : "memory");
    } else {
      // this CTA's part of x: codes in the MMA's 128-byte swizzle, scales beside them; a half-warp per row and K block
      const int hw = fw * 2 + (lane >> 4), hl = lane & 15;
      const int items = kbs * rows;
      for (int base = 0; base < items; base += 64) {
        uint4 u[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = base + 16 * j + hw;
          u[j] = make_uint4(0, 0, 0, 0);
          if (i < items) {
            const int kb = i / rows, r = i - kb * rows, col = (kb0 + kb) * BK + hl * 8;
            if (col < p.K) u[j] = *reinterpret_cast<const uint4*>(p.x + (int64_t)(row0 + r) * p.ldx + col);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (base + 16 * j >= items) break;  // the whole CTA alike
          const int i = base + 16 * j + hw;
          uint2 q;
          float s;
          quant8(u[j], p.fp16 != 0, p.pow2 != 0, q, s);
          if (i < items) {
            const int kb = i / rows, r = i - kb * rows;
            *reinterpret_cast<uint2*>(sX + kb * TN * BK + r * 128 + (((hl >> 1) ^ (r & 7)) << 4) + (hl & 1) * 8) = q;
            if (hl == 0) sSa[kb * TN + r] = s;
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(x_full);
    }
    // ---------------- fold: acc[c] += partial[c] * (sa[token c] * sb)
    const int quarter = warp & 3, part = fw >> 2;
    const int tok0 = SWIGLU ? 0 : part * C;
    const uint32_t t_lane = tmem_base + ((uint32_t)(quarter * 32) << 16) + part * C;
    float acc[C];
#pragma unroll
    for (int i = 0; i < C; ++i) acc[i] = 0.f;
    // G columns are loaded while the G before them are folded, across K blocks as well.  The factors are there: all eight
    // warps have written theirs (XTMA: behind the bar.sync, else before the MMAs started).
    constexpr int G = T::G, CHUNKS = C / G;
    static_assert(CHUNKS <= 2, "two chunks, or one");
    uint32_t va[G], vb[G];
    ok = warp_wait(&acc_full[0], 0, abort_flag);
    tc_fence_after();
    if (ok) tmem_ld_cols(t_lane, va);
    for (int i = 0; ok && i < kbs; ++i) {
      const uint32_t buf = i % T::BUFS, next = (i + 1) % T::BUFS, next_parity = ((i + 1) / T::BUFS) & 1u;
      const bool more = i + 1 < kbs;
      const float sb = sSb[2 * i + (SWIGLU ? part : 0)];
      const float* sa = sSa + i * TN + tok0;
      const bool early = more && mbar_try_wait(&acc_full[next], next_parity);
      tmem_wait_cols(va);
      if constexpr (CHUNKS == 2) {
        tmem_ld_cols(t_lane + buf * T::ACC_COLS + G, vb);
        fold_cols(acc, va, sa, sb);
        tmem_wait_cols(vb);
      }
      tc_fence_before();  // the buffer has been read
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[buf]);
      if (more) {
        if (!__all_sync(0xffffffffu, early)) ok = warp_wait(&acc_full[next], next_parity, abort_flag);
        tc_fence_after();
      }
      if constexpr (CHUNKS == 2) {
        if (more && ok) tmem_ld_cols(t_lane + next * T::ACC_COLS, va);
        fold_cols(acc + G, vb, sa + G, sb);
      } else {
        if (more && ok) tmem_ld_cols(t_lane + next * T::ACC_COLS, vb);
        fold_cols(acc, va, sa, sb);
        tmem_wait_cols(vb);
#pragma unroll
        for (int c = 0; c < G; ++c) va[c] = vb[c];
      }
    }
    // every MMA that read a stage has completed, this warp waited for its partial: the tile may take the stages' place
    if (ok) {
      float* part_out = reinterpret_cast<float*>(sW) + (part * C) * 128 + quarter * 32 + lane;
#pragma unroll
      for (int i = 0; i < C; ++i) part_out[i * 128] = acc[i];
    }
  }
  grid_dependents_launch();
  __syncwarp();
  cluster_sync();

  // ---------------- the cluster's partials, added in rank order
  const uint32_t base = smem_u32(sW);
  if (*abort_flag) {  // copies may still be on their way into this block's shared memory: let them land before it ends
    if (threadIdx.x == 0) report(p.status, status_word(ASAP_ST_PIPELINE_TIMEOUT, 0, 0, 18 + SWIGLU));
    const uint64_t landed = globaltimer_ns() + 200000000ull;
    while (globaltimer_ns() < landed) {
    }
    __syncwarp();
  } else {
    if constexpr (!SWIGLU) {
      const int quads = 32 / S;  // this CTA's share of the tile's 32 groups of 4 columns
      for (int i = threadIdx.x; i < rows * quads; i += SK_THREADS) {
        const int r = i / quads, c = (rank * quads + i - r * quads) * 4;
        const float4 a = cluster_sum(base + (r * 128 + c) * 4, S);
        if (n_t * 128 + c < p.N) {
          uint16_t* o = reinterpret_cast<uint16_t*>(p.out) + (int64_t)(row0 + r) * p.N + n_t * 128 + c;
          *reinterpret_cast<uint2*>(o) = make_uint2(pack16(a.x, a.y, p.fp16 != 0), pack16(a.z, a.w, p.fp16 != 0));
        }
      }
    } else {
      for (int r = rank + S * warp; r < rows; r += S * (SK_THREADS / 32)) {  // a warp per row, 4 columns per lane
        const float4 g = cluster_sum(base + (r * 128 + 4 * lane) * 4, S);
        const float4 u = cluster_sum(base + ((TN + r) * 128 + 4 * lane) * 4, S);
        const float lim = p.swiglu_limit;
        const float h[4] = {swiglu(g.x, u.x, lim), swiglu(g.y, u.y, lim), swiglu(g.z, u.z, lim), swiglu(g.w, u.w, lim)};
        float amax = fmaxf(fmaxf(fabsf(h[0]), fabsf(h[1])), fmaxf(fabsf(h[2]), fabsf(h[3])));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        float scale, inv;
        block_scale(amax, p.pow2 != 0, scale, inv);
        *reinterpret_cast<uint32_t*>(p.out_q + (int64_t)(row0 + r) * (p.N / 2) + n_t * 128 + 4 * lane) = codes4(h, inv);
        if (lane == 0) p.out_sa[(int64_t)n_t * p.mp + row0 + r] = scale;
      }
    }
  }
  tc_fence_before();
  cluster_leave();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, T::TMEM);
  }
}

}  // namespace lin
