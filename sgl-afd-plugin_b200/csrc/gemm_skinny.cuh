// FP8 block-scaled linear for few rows: the weight tile is the MMA's 128-row operand, the rows of x its TN columns, and
// the K blocks of a tile are split over a cluster of S CTAs.  Included by linear.cu.
//
// With few rows the cost is reading the weights once, and the launch.  So one launch does it all: every CTA quantises
// the part of x that its K blocks need itself (a few KB, from L2) while TMA already fetches its weights, and the
// cluster adds its S partial tiles through distributed shared memory in rank order: no scratch in memory, no second
// kernel, the same bits every time.  Splitting K makes 128 to 300 CTAs of a product that has 16 to 56 weight tiles, and
// puts most of a CTA's weights in flight at once.
#pragma once

namespace lin {

constexpr int SK_FOLD_WARPS = 8, SK_THREADS = 32 * (2 + SK_FOLD_WARPS);
constexpr int SK_MAX_KB = 64, SK_MAX_STAGES = 12, SK_MAX_SPLIT = 8;

template <int TN, int SWIGLU>
struct Skinny {
  static constexpr int TILES = SWIGLU ? 2 : 1;          // weight tiles of 128 rows per CTA (gate and up)
  static constexpr int STAGE_BYTES = TILES * 128 * BK;
  static constexpr int ACC_COLS = TILES * TN;           // TMEM columns of one K block's partial
  static constexpr int BUFS = 256 / ACC_COLS;           // 256 columns, so that two CTAs fit an SM
  static constexpr int C = ACC_COLS / 2;                // columns per folding warp
  static_assert(BUFS >= 2, "two partials at least");
};

struct SkinnyParams {
  CUtensorMap tmap_w;  // weights [N, K]
  const uint16_t* x;
  int64_t ldx;
  int32_t M, K, N, KB, NB, split, stages, max_kb;
  const float* sb;
  int32_t fp16, pow2;
  void* out;  // linear: [M, N] of x's type
  float swiglu_limit;
  uint8_t* out_q;  // SwiGLU: codes of h [M, N / 2]
  float* out_sa;   // SwiGLU: scales of h [N / 256][mp]
  int64_t mp;
  // the rows may come quantised already (the second product of the shared expert)
  const uint8_t* xq;  // codes [M, 128 KB] or NULL
  const float* sa;    // scales [KB][mp]
  uint64_t status, timeout_ns;
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 peer_load4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
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

template <int TN, int SWIGLU>
__global__ void __launch_bounds__(SK_THREADS, Skinny<TN, SWIGLU>::C <= 32 ? 2 : 1)
    linear_skinny_kernel(const __grid_constant__ SkinnyParams p) {
  using T = Skinny<TN, SWIGLU>;
  constexpr int C = T::C;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sW = smem;                                   // [stages][TILES][128 rows x 128 B]
  uint8_t* sX = sW + p.stages * T::STAGE_BYTES;         // [max_kb][TN rows x 128 B]
  float* sSa = reinterpret_cast<float*>(sX + p.max_kb * TN * BK);  // [max_kb][TN]
  float* sSb = sSa + p.max_kb * TN;                     // [max_kb][2]
  uint64_t* full = reinterpret_cast<uint64_t*>(sSb + 2 * p.max_kb);
  uint64_t* empty = full + SK_MAX_STAGES;
  uint64_t* x_full = empty + SK_MAX_STAGES;  // [max_kb <= SK_MAX_KB]
  uint64_t* acc_full = x_full + SK_MAX_KB;   // [BUFS <= 16]
  uint64_t* acc_empty = acc_full + 16;
  uint64_t* mma_done = acc_empty + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank(), S = p.split;
  const int n_t = blockIdx.x / S;
  const int row0 = blockIdx.y * TN, rows = min(TN, p.M - row0);
  const int kb0 = rank * p.KB / S, kbs = (rank + 1) * p.KB / S - kb0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < kbs; ++i) mbar_init(&x_full[i], SK_FOLD_WARPS);
    for (int b = 0; b < T::BUFS; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], SK_FOLD_WARPS);
    }
    mbar_init(mma_done, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 256);
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
      int stage = 0;
      uint32_t phase = 0;
      int issued = 0;
      for (int i = 0; i < kbs; ++i) {
        ok = mbar_wait(&empty[stage], phase ^ 1u, deadline, abort_flag);
        if (!ok) break;
        uint8_t* dst = sW + stage * T::STAGE_BYTES;
        mbar_arrive_expect_tx(&full[stage], T::STAGE_BYTES);
        tma_load_2d(dst, &p.tmap_w, (kb0 + i) * BK, b0, &full[stage]);
        if constexpr (SWIGLU) tma_load_2d(dst + 128 * BK, &p.tmap_w, (kb0 + i) * BK, b1, &full[stage]);
        ++issued;
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) {  // copies in flight must land before this CTA may exit (else an MMA has waited for each)
        const uint64_t drain_deadline = globaltimer_ns() + 200000000ull;
        volatile int no_abort = 0;
        for (int i = 0; i < min(issued, p.stages); ++i) {
          int s = stage - 1 - i;
          uint32_t ph = phase;
          if (s < 0) {
            s += p.stages;
            ph ^= 1u;
          }
          mbar_wait(&full[s], ph, drain_deadline, &no_abort);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_f8f6f4(128, TN);
      int stage = 0;
      uint32_t phase = 0;
      for (int i = 0; i < kbs; ++i) {
        const uint32_t buf = i % T::BUFS;
        ok = mbar_wait(&acc_empty[buf], ((i / T::BUFS) & 1u) ^ 1u, deadline, abort_flag) &&
             mbar_wait(&x_full[i], 0, deadline, abort_flag) && mbar_wait(&full[stage], phase, deadline, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint64_t wdesc = sdesc_sw128(sW + stage * T::STAGE_BYTES), xdesc = sdesc_sw128(sX + i * TN * BK);
#pragma unroll
        for (int h = 0; h < T::TILES; ++h)
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            tc_mma_f8f6f4(tmem_base + buf * T::ACC_COLS + h * TN, wdesc + (uint64_t)(h * 128 * BK >> 4) + 2ull * k,
                          xdesc + 2ull * k, idesc, k != 0);
        tc_commit(&empty[stage]);
        tc_commit(&acc_full[buf]);
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      tc_commit(mma_done);
      volatile int no_abort = 0;
      mbar_wait(mma_done, 0, globaltimer_ns() + 200000000ull, &no_abort);
    }
  } else {
    // ---------------- this CTA's part of x: codes in the MMA's 128-byte swizzle, scales beside them
    const int fw = warp - 2, hw = fw * 2 + (lane >> 4), hl = lane & 15;
    for (int i = threadIdx.x - 64; i < kbs; i += 32 * SK_FOLD_WARPS) {
      const int nb1 = p.NB / 2 + n_t;
      sSb[2 * i] = __ldg(p.sb + (int64_t)n_t * p.KB + kb0 + i);
      sSb[2 * i + 1] = SWIGLU ? __ldg(p.sb + (int64_t)nb1 * p.KB + kb0 + i) : 0.f;
    }
    const int items = kbs * rows;
    int done_kb = 0;
    for (int base = 0; base < items; base += 64) {
      uint4 u[4];
      uint2 q[4];
      float s[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = base + 16 * j + hw;
        u[j] = make_uint4(0, 0, 0, 0);
        q[j] = make_uint2(0, 0);
        s[j] = 0.f;
        if (i < items) {
          const int kb = i / rows, r = i - kb * rows, col = (kb0 + kb) * BK + hl * 8;
          if (p.xq) {
            q[j] = *reinterpret_cast<const uint2*>(p.xq + (int64_t)(row0 + r) * p.KB * BK + col);
            s[j] = p.sa[(int64_t)(kb0 + kb) * p.mp + row0 + r];
          } else if (col < p.K) {
            u[j] = *reinterpret_cast<const uint4*>(p.x + (int64_t)(row0 + r) * p.ldx + col);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = base + 16 * j + hw;
        if (!p.xq) quant8(u[j], p.fp16 != 0, p.pow2 != 0, q[j], s[j]);
        if (i < items) {
          const int kb = i / rows, r = i - kb * rows;
          *reinterpret_cast<uint2*>(sX + kb * TN * BK + r * 128 + (((hl >> 1) ^ (r & 7)) << 4) + (hl & 1) * 8) = q[j];
          if (hl == 0) sSa[kb * TN + r] = s[j];
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      // this warp has written every item below base + 64 that is its own
      const int upto = base + 64 >= items ? kbs : (base + 64) / rows;
      if (lane == 0)
        for (int kb = done_kb; kb < upto; ++kb) mbar_arrive(&x_full[kb]);
      done_kb = upto;
    }
    // ---------------- fold: acc[c] += partial[c] * (sa[token c] * sb)
    const int quarter = warp & 3, part = fw >> 2;
    const int tok0 = SWIGLU ? 0 : part * C;
    const uint32_t t_lane = tmem_base + ((uint32_t)(quarter * 32) << 16) + part * C;
    float acc[C];
#pragma unroll
    for (int i = 0; i < C; ++i) acc[i] = 0.f;
    for (int i = 0; i < kbs; ++i) {
      const uint32_t buf = i % T::BUFS;
      ok = warp_wait(&x_full[i], 0, abort_flag) &&
           warp_wait(&acc_full[buf], (i / T::BUFS) & 1u, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const float sb = sSb[2 * i + (SWIGLU ? part : 0)];
      const float* sa = sSa + i * TN + tok0;
      constexpr int G = C < 32 ? C : 32;
#pragma unroll
      for (int c0 = 0; c0 < C; c0 += G) {
        uint32_t v[32];
        const uint32_t ta = t_lane + buf * T::ACC_COLS + c0;
        if constexpr (G == 8) tmem_ld_32x32b_x8(ta, v);
        else if constexpr (G == 16) tmem_ld_32x32b_x16(ta, v);
        else tmem_ld_32x32b_x32(ta, v);
        tmem_wait_ld();
        if (c0 + G == C) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_empty[buf]);
        }
#pragma unroll
        for (int c = 0; c < G; c += 4) {
          const float4 f = *reinterpret_cast<const float4*>(sa + c0 + c);
          acc[c0 + c] = fmaf(__uint_as_float(v[c]), f.x * sb, acc[c0 + c]);
          acc[c0 + c + 1] = fmaf(__uint_as_float(v[c + 1]), f.y * sb, acc[c0 + c + 1]);
          acc[c0 + c + 2] = fmaf(__uint_as_float(v[c + 2]), f.z * sb, acc[c0 + c + 2]);
          acc[c0 + c + 3] = fmaf(__uint_as_float(v[c + 3]), f.w * sb, acc[c0 + c + 3]);
        }
      }
    }
    // every MMA that read a stage has completed, this warp waited for its partial: the tile may take the stages' place
    if (ok) {
      float* part_out = reinterpret_cast<float*>(sW) + (part * C) * 128 + quarter * 32 + lane;
#pragma unroll
      for (int i = 0; i < C; ++i) part_out[i * 128] = acc[i];
    }
  }
  __syncwarp();
  cluster_sync();

  // ---------------- the cluster's partials, added in rank order
  const uint32_t base = smem_u32(sW);
  if (*abort_flag) {
    if (threadIdx.x == 0) report(p.status, status_word(ASAP_ST_PIPELINE_TIMEOUT, 0, 0, 18 + SWIGLU));
  } else {
    if constexpr (!SWIGLU) {
      const int quads = 32 / S;  // this CTA's share of the tile's 32 groups of 4 columns
      for (int i = threadIdx.x; i < rows * quads; i += SK_THREADS) {
        const int r = i / quads, c = (rank * quads + i - r * quads) * 4;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s = 0; s < S; ++s) {
          const float4 v = peer_load4(peer_addr(base + (r * 128 + c) * 4, s));
          a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
        }
        if (n_t * 128 + c < p.N) {
          uint16_t* o = reinterpret_cast<uint16_t*>(p.out) + (int64_t)(row0 + r) * p.N + n_t * 128 + c;
          *reinterpret_cast<uint2*>(o) = make_uint2(pack16(a.x, a.y, p.fp16 != 0), pack16(a.z, a.w, p.fp16 != 0));
        }
      }
    } else {
      for (int r = rank + S * warp; r < rows; r += S * (SK_THREADS / 32)) {  // a warp per row, 4 columns per lane
        float4 g = make_float4(0.f, 0.f, 0.f, 0.f), u = g;
        for (int s = 0; s < S; ++s) {
          const float4 a = peer_load4(peer_addr(base + (r * 128 + 4 * lane) * 4, s));
          const float4 b = peer_load4(peer_addr(base + ((TN + r) * 128 + 4 * lane) * 4, s));
          g.x += a.x, g.y += a.y, g.z += a.z, g.w += a.w;
          u.x += b.x, u.y += b.y, u.z += b.z, u.w += b.w;
        }
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
  cluster_sync();  // no CTA leaves while another reads its shared memory
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 256);
  }
}

}  // namespace lin
