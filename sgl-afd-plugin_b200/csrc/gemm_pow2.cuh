// FP8 linear whose scales are all powers of two (E8M0): they ride in the MMA (kind::mxf8f6f4.block_scale), the
// accumulator stays in TMEM over all of K, and nothing is folded.  Included by linear.cu.
//
// Same tiles, order and epilogues as linear_gemm_kernel.  Scales travel as atoms of 512 bytes (128 rows x four blocks of
// 32 along K; byte (row % 32) * 16 + (row / 32) * 4 + k-block), which tcgen05.cp spreads over the TMEM lanes.  A block of
// 128 along K has one scale, so the four bytes of a row are the same; a weight atom is one byte 512 times, laid out once
// with the weight.
#pragma once

namespace lin {

constexpr int ATOM = 512;
constexpr int P2_STAGE_BYTES = A_BYTES + B_BYTES + 3 * ATOM;
constexpr int P2_EPI_BASE = 2, P2_THREADS = 32 * (P2_EPI_BASE + EPI_WARPS);
constexpr int P2_SMEM_BYTES = 1024 + STAGES * P2_STAGE_BYTES + STAGE_OUT_BYTES + CTRL_BYTES;
static_assert(P2_SMEM_BYTES <= 232448, "shared memory over the 227 KB per block");
constexpr uint32_t P2_SFA = 256, P2_SFB = 256 + 4 * STAGES;  // TMEM columns behind the accumulator's 256
static_assert(P2_SFB + 8 * STAGES <= TMEM_COLS, "scale columns over tensor memory");

// kind::mxf8f6f4: A = B = E4M3, K-major, UE8M0 scales
__host__ __device__ constexpr uint32_t idesc_mxf8(int M, int N) {
  return ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ uint64_t sdesc_atom(const void* p) {
  const uint64_t a = smem_u32(p);
  return ((a >> 4) & 0x3FFFull) | (1ull << 16) | ((uint64_t)(128 >> 4) << 32) | (1ull << 46);
}
// Byte offset of a row's scales for K block kb (of 128) among KB: one word, the byte four times.
__host__ __device__ constexpr int64_t atom_off(int64_t row, int kb, int KB) {
  return ((row >> 7) * KB + kb) * ATOM + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}
__device__ __forceinline__ uint32_t atom_word(float pow2_scale) {
  return (__float_as_uint(pow2_scale) >> 23) * 0x01010101u;
}

template <int SWIGLU, bool SPLIT = false>
__global__ void __launch_bounds__(P2_THREADS, 1) linear_pow2_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + STAGES * A_BYTES;
  uint8_t* sSF = sB + STAGES * B_BYTES;  // [STAGES][A atom, two B atoms]
  uint8_t* sOut = sSF + STAGES * 3 * ATOM;
  uint8_t* ctrl = sOut + STAGE_OUT_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(ctrl);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + 1;
  uint64_t* mma_done = acc_empty + 1;
  uint64_t* amax_bar = mma_done + 1;  // [4 lane quarters][2 tile parities]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ctrl + 512);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(ctrl + 516);
  float* s_amax = reinterpret_cast<float*>(ctrl + 1024);  // [2 tile parities][2 halves][128 rows]

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, EPI_WARPS);
    mbar_init(mma_done, 1);
    for (int b = 0; b < 8; ++b) mbar_init(&amax_bar[b], 64);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&p.tmap_a);
    prefetch_tmap(&p.tmap_b);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int num_tiles = p.m_tiles * p.n_tiles;
  // with split > 1 a cluster has one tile, and this CTA the K blocks [kb0, kb0 + KB) of it
  const int split = SPLIT ? p.split : 1, rank = SPLIT ? (int)cluster_rank() : 0;
  const int kb0 = rank * p.KB / split, KB = (rank + 1) * p.KB / split - kb0;
  const int tile0 = blockIdx.x / split, tile_step = gridDim.x / split;
  const uint64_t deadline = globaltimer_ns() + p.timeout_ns;

  if (warp == 0) {
    // ---------------- TMA producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = tile0; ok && tile < num_tiles; tile += tile_step) {
        int m_t, n_t;
        decode_tile(p, tile, m_t, n_t);
        const int b0 = SWIGLU ? n_t * 128 : n_t * BN, b1 = SWIGLU ? p.N / 2 + n_t * 128 : n_t * BN + 128;
        const uint8_t* sfa = p.sfa + ((int64_t)m_t * p.KB + kb0) * ATOM;
        const uint8_t* sfb0 = p.sfb + ((int64_t)kb0 * p.nb_atoms + b0 / 128) * ATOM;
        const uint8_t* sfb1 = p.sfb + ((int64_t)kb0 * p.nb_atoms + b1 / 128) * ATOM;
        for (int kb = 0; kb < KB; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, deadline, abort_flag)) {
            ok = false;
            break;
          }
          uint8_t* sf = sSF + stage * 3 * ATOM;
          mbar_arrive_expect_tx(&full[stage], P2_STAGE_BYTES);
          tma_load_2d(sA + stage * A_BYTES, &p.tmap_a, (kb0 + kb) * BK, m_t * BM, &full[stage]);
          tma_load_2d(sB + stage * B_BYTES, &p.tmap_b, (kb0 + kb) * BK, b0, &full[stage]);
          tma_load_2d(sB + stage * B_BYTES + B_HALF, &p.tmap_b, (kb0 + kb) * BK, b1, &full[stage]);
          bulk_load(sf, sfa + (int64_t)kb * ATOM, ATOM, &full[stage]);
          bulk_load(sf + ATOM, sfb0 + (int64_t)kb * p.nb_atoms * ATOM, ATOM, &full[stage]);
          bulk_load(sf + 2 * ATOM, sfb1 + (int64_t)kb * p.nb_atoms * ATOM, ATOM, &full[stage]);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer
    int stage = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool ok = true;
    for (int tile = tile0; ok && tile < num_tiles; tile += tile_step) {
      ok = __all_sync(0xffffffffu, mbar_wait(acc_empty, acc_phase ^ 1u, deadline, abort_flag));
      if (!ok) break;
      for (int kb = 0; kb < KB; ++kb) {
        const uint64_t adesc = sdesc_sw128(sA + stage * A_BYTES), bdesc = sdesc_sw128(sB + stage * B_BYTES);
        const uint8_t* sf = sSF + stage * 3 * ATOM;
        const uint32_t t_sfa = tmem_base + P2_SFA + 4 * stage, t_sfb = tmem_base + P2_SFB + 8 * stage;
        ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], phase, deadline, abort_flag));
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          tc_cp_32x128b_warpx4(t_sfa, sdesc_atom(sf));
          tc_cp_32x128b_warpx4(t_sfb, sdesc_atom(sf + ATOM));
          tc_cp_32x128b_warpx4(t_sfb + 4, sdesc_atom(sf + 2 * ATOM));
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            tc_mma_mxf8f6f4(tmem_base, adesc + 2ull * k, bdesc + 2ull * k, idesc_mxf8(BM, BN), (kb | k) != 0, t_sfa,
                            t_sfb);
          tc_commit(&empty[stage]);
          if (kb + 1 == KB) tc_commit(acc_full);
        }
        __syncwarp();
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
      acc_phase ^= 1u;
    }
    if (elect_one()) tc_commit(mma_done);
    __syncwarp();
    drain_mmas(mma_done, deadline, abort_flag);
  } else {
    // ---------------- epilogue
    const int q = warp & 3;                      // TMEM lane quarter this warp may access
    const int half = (warp - P2_EPI_BASE) >> 2;  // which half of the tile's columns
    const uint32_t t_lane = tmem_base + ((uint32_t)(q * 32) << 16);
    const int col0 = SWIGLU ? 64 * half : 128 * half;
    const int col1 = SWIGLU ? 128 + 64 * half : 128 * half + 64;
    uint32_t tcount = 0;
    bool exchanged = false;
    for (int tile = tile0; tile < num_tiles; tile += tile_step, ++tcount) {
      int m_t, n_t;
      decode_tile(p, tile, m_t, n_t);
      if (!warp_wait(acc_full, tcount & 1u, abort_flag)) break;
      tc_fence_after();
      uint32_t v[4][32];
      tmem_ld_32x32b_x32(t_lane + col0, v[0]);
      tmem_ld_32x32b_x32(t_lane + col0 + 32, v[1]);
      tmem_ld_32x32b_x32(t_lane + col1, v[2]);
      tmem_ld_32x32b_x32(t_lane + col1 + 32, v[3]);
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_wait_regs(v[c]);
      tc_fence_before();  // the accumulator is in registers: the next tile's MMAs may start
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty);
      const int row0 = m_t * BM + q * 32;
      if constexpr (SWIGLU) {
        float amax = 0.f, h[64];
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          h[i] = swiglu(__uint_as_float(v[i / 32][i % 32]), __uint_as_float(v[2 + i / 32][i % 32]), p.swiglu_limit);
          amax = fmaxf(amax, fabsf(h[i]));
        }
        // the row's other 64 h values live in the partner warp (same lane quarter, other half)
        const uint32_t par = tcount & 1u;
        const int row_in_tile = q * 32 + lane;
        s_amax[(par * 2 + half) * 128 + row_in_tile] = amax;
        mbar_arrive(&amax_bar[q * 2 + par]);
        if (!warp_wait(&amax_bar[q * 2 + par], (tcount >> 1) & 1u, abort_flag)) break;
        amax = fmaxf(amax, s_amax[(par * 2 + (half ^ 1)) * 128 + row_in_tile]);
        if (row0 + lane < p.M) {
          float scale, inv;
          block_scale(amax, true, scale, inv);
          uint4* dst = reinterpret_cast<uint4*>(p.out_q + (int64_t)(row0 + lane) * (p.N / 2) + n_t * 128 + half * 64);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            dst[j] = make_uint4(codes4(h + 16 * j, inv), codes4(h + 16 * j + 4, inv), codes4(h + 16 * j + 8, inv),
                                codes4(h + 16 * j + 12, inv));
          if (half == 0)
            *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(p.out_sa) +
                                         atom_off(row0 + lane, n_t, p.N / 256)) = atom_word(scale);
        }
      } else {
        uint64_t a0[32], a1[32];  // pairs of columns
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          a0[i] = pair(__uint_as_float(v[i / 16][2 * (i % 16)]), __uint_as_float(v[i / 16][2 * (i % 16) + 1]));
          a1[i] = pair(__uint_as_float(v[2 + i / 16][2 * (i % 16)]), __uint_as_float(v[2 + i / 16][2 * (i % 16) + 1]));
        }
        if constexpr (SPLIT) {  // the partials take the place of the operands, which every MMA is done with
          exchange(a0, a1, reinterpret_cast<float*>(sA), split, rank, half, q * 32 + lane, true);
          exchanged = true;
        }
        uint8_t* wb = sOut + (warp - P2_EPI_BASE) * 2048;
        const int c0 = n_t * BN + half * 128;
        uint16_t* out0 = reinterpret_cast<uint16_t*>(p.out) + (int64_t)row0 * p.ldo + c0;
        const bool fp16 = p.out_fp16 != 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (SPLIT && !finishes(split, rank, half, c / 2)) continue;
          const uint64_t* a = c < 2 ? a0 + 16 * c : a1 + 16 * (c - 2);
          uint32_t o[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 f = halves(a[i]);
            o[i] = pack16(f.x, f.y, fp16);
          }
          store_rows(o, wb, out0 + 32 * c, p.ldo, p.M - row0, p.N - c0 - 32 * c, lane);
        }
      }
    }
    if (SPLIT && !exchanged) {  // this warp gave up: the cluster's barrier still counts it
      __syncwarp();
      cluster_sync();
    }
  }
  if constexpr (SPLIT) {
    __syncwarp();
    if (warp < P2_EPI_BASE) cluster_sync();  // the exchange's barrier
    cluster_leave();
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {  // copies may still be on their way into this block's shared memory: let them land before it ends
    if (threadIdx.x == 0) report(p.status, status_word(ASAP_ST_PIPELINE_TIMEOUT, 0, 0, 20 + SWIGLU));
    const uint64_t landed = globaltimer_ns() + 200000000ull;
    while (globaltimer_ns() < landed) {
    }
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

}  // namespace lin
