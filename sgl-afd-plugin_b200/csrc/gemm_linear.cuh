// FP8 block-scaled linear, y = deq(xq) deq(W)^T: tiles of 128 rows x 256 weight rows on tcgen05 kind::f8f6f4.
// Included by linear.cu.
//
// y[r][n] = sum_kb sa[r][kb] * sb[n / 128][kb] * sum_{k in block kb} xq[r][k] * w[n][k].  fp32 scales are not powers
// of two and cannot ride in the MMA, so every 128-deep K block is accumulated on its own into one of two TMEM buffers
// and folded into fp32 registers (one fma per element) while the tensor core fills the other buffer.
//
// A probe of the fold alone (148 SMs, operands fixed in shared memory) runs one K block of 128 x 256 in 390 cycles,
// and with the MMAs and their hand-over in 640, against 512 for the MMAs by themselves.  What keeps a kernel from
// that is a global load on the fold's path: so one warp multiplies the two scales of each row and K block ahead of
// time into a ring of shared-memory slots (kScaleSlots K blocks, about 4 K cycles, deep) and the fold reads one word.
#pragma once

namespace lin {

constexpr int BM = 128, BN = 256, BK = 128;
constexpr int STAGES = 4;
constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK, B_HALF = B_BYTES / 2;
constexpr uint32_t STAGE_TX = A_BYTES + B_BYTES;
constexpr int kScaleSlots = 8;
constexpr int SCALE_BYTES = 2 * BM * 4;  // a K block's factor per row, one set per 128 weight rows of the tile
constexpr int EPI_WARPS = 8, EPI_BASE = 4, THREADS = 32 * (EPI_BASE + EPI_WARPS);
constexpr uint32_t TMEM_COLS = 512;
constexpr int STAGE_OUT_BYTES = EPI_WARPS * 2048;
constexpr int CTRL_BYTES = 4096;  // barriers, TMEM slot, row amax exchange
constexpr int SMEM_BYTES =
    1024 + STAGES * (A_BYTES + B_BYTES) + kScaleSlots * SCALE_BYTES + STAGE_OUT_BYTES + CTRL_BYTES;
static_assert(SMEM_BYTES <= 232448, "shared memory over the 227 KB per block");
// m-tiles that share a pass over the weight tiles: 16 x 9 tiles are in flight on 148 SMs, so a K block of both
// operands is read from L2 about 12 times per 128-row tile whatever M and N are.
constexpr int GROUP_M = 16;

struct Params {
  CUtensorMap tmap_a;  // activation codes [M, K], rows K padded to 128 apart
  CUtensorMap tmap_b;  // weights [N, K]
  const float* sa;     // activation scales [K blocks][mp]
  const float* sb;     // weight scales [N blocks][K blocks]
  int64_t mp;          // M rounded up to 128
  int32_t M, N, KB, NB, m_tiles, n_tiles;
  void* out;           // linear: [M, N], bf16 or fp16
  int64_t ldo;
  int32_t out_fp16;
  float swiglu_limit;  // SwiGLU: N = 2I, gate rows then up rows
  uint8_t* out_q;      // SwiGLU: codes of h [M, I]
  float* out_sa;       // SwiGLU: scales of h [I / 128][mp]
  int32_t pow2;        // scales of h are powers of two
  uint64_t status, timeout_ns;
};

__host__ __device__ constexpr uint32_t idesc_f8f6f4(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// K-major, 128-byte swizzle, 8-row groups 1024 bytes apart
__device__ __forceinline__ uint64_t sdesc_sw128(const void* p) {
  const uint64_t a = smem_u32(p);
  return ((a >> 4) & 0x3FFFull) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// A bounded wait of a whole warp: every lane gets the same answer and the warp is converged after it.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, uint64_t deadline, volatile int* abort) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, deadline, abort));
}

// acc[i] += x[i] * f, two per instruction
__device__ __forceinline__ void fold32(float* acc, const uint32_t (&x)[32], float f) {
  const float2 ff = make_float2(f, f);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float2 r = __ffma2_rn(make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), ff,
                                make_float2(acc[2 * i], acc[2 * i + 1]));
    acc[2 * i] = r.x;
    acc[2 * i + 1] = r.y;
  }
}

__device__ __forceinline__ void decode_tile(const Params& p, int tile, int& m_t, int& n_t) {
  const int per_group = GROUP_M * p.n_tiles;
  const int g = tile / per_group, local = tile - g * per_group;
  const int gm = min(GROUP_M, p.m_tiles - g * GROUP_M);
  n_t = local / gm;
  m_t = g * GROUP_M + local % gm;
}

__device__ __forceinline__ uint32_t pack16(float a, float b, bool fp16) {
  if (fp16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A warp's 32 rows x 32 16-bit values (lane = row) through its 2 KB buffer, so that a store instruction writes 8 rows
// x 64 contiguous bytes; 16-byte units XOR-swizzled by (row >> 1) & 3 keep both sides free of bank conflicts.
__device__ __forceinline__ void store_rows(const uint32_t (&o)[16], uint8_t* wb, uint16_t* out0, int64_t ldo,
                                           int rows_left, int cols_left, int lane) {
  uint4* mine = reinterpret_cast<uint4*>(wb + lane * 64);
#pragma unroll
  for (int u = 0; u < 4; ++u)
    mine[u ^ ((lane >> 1) & 3)] = make_uint4(o[4 * u], o[4 * u + 1], o[4 * u + 2], o[4 * u + 3]);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = i * 8 + (lane >> 2), u = lane & 3;
    const uint4 v = reinterpret_cast<const uint4*>(wb + row * 64)[u ^ ((row >> 1) & 3)];
    if (row < rows_left && 8 * u < cols_left) *reinterpret_cast<uint4*>(out0 + row * ldo + u * 8) = v;
  }
  __syncwarp();
}

// SWIGLU 0: out = the tile, 16 bit.  SWIGLU 1: tile n covers gate rows [128n, 128n + 128) and up rows I further;
// h = silu(gate) * up, requantised per 1 x 128 (the tile's 128 h columns are one K block of the down product).
template <int SWIGLU>
__global__ void __launch_bounds__(THREADS, 1) linear_gemm_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + STAGES * A_BYTES;
  float* sF = reinterpret_cast<float*>(sB + STAGES * B_BYTES);  // [kScaleSlots][2][BM]
  uint8_t* sOut = reinterpret_cast<uint8_t*>(sF) + kScaleSlots * SCALE_BYTES;
  uint8_t* ctrl = sOut + STAGE_OUT_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(ctrl);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;         // [2]
  uint64_t* acc_empty = acc_full + 2;          // [2]
  uint64_t* sc_full = acc_empty + 2;           // [kScaleSlots]
  uint64_t* sc_empty = sc_full + kScaleSlots;  // [kScaleSlots]
  uint64_t* mma_done = sc_empty + kScaleSlots;
  uint64_t* amax_bar = mma_done + 1;  // [4 lane quarters][2 tile parities]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ctrl + 512);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(ctrl + 516);
  float* s_amax = reinterpret_cast<float*>(ctrl + 1024);  // [2 tile parities][2 halves][128 rows]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], EPI_WARPS);
    }
    for (int s = 0; s < kScaleSlots; ++s) {
      mbar_init(&sc_full[s], 1);
      mbar_init(&sc_empty[s], EPI_WARPS);
    }
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
  const int KB = p.KB;
  const int num_tiles = p.m_tiles * p.n_tiles;
  const uint64_t deadline = globaltimer_ns() + p.timeout_ns;

  // Registers (as launched 384 x 168 = 64512): the four helper warps give theirs up, the folding warps hold the
  // 128 accumulators and two TMEM loads in flight: 128 x 48 + 256 x 224 = 63488.
  if (warp < EPI_BASE) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 48;\n" ::: "memory");
    if (warp == 0) {
      // ---------------- TMA producer
      if (lane == 0) {
        int stage = 0, issued = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int tile = blockIdx.x; ok && tile < num_tiles; tile += gridDim.x) {
          int m_t, n_t;
          decode_tile(p, tile, m_t, n_t);
          const int b0 = SWIGLU ? n_t * 128 : n_t * BN, b1 = SWIGLU ? p.N / 2 + n_t * 128 : n_t * BN + 128;
          for (int kb = 0; kb < KB; ++kb) {
            if (!mbar_wait(&empty[stage], phase ^ 1u, deadline, abort_flag)) {
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(&full[stage], STAGE_TX);
            tma_load_2d(sA + stage * A_BYTES, &p.tmap_a, kb * BK, m_t * BM, &full[stage]);
            tma_load_2d(sB + stage * B_BYTES, &p.tmap_b, kb * BK, b0, &full[stage]);
            tma_load_2d(sB + stage * B_BYTES + B_HALF, &p.tmap_b, kb * BK, b1, &full[stage]);
            ++issued;
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
        // the copies of the last armed stages must land before this CTA may exit
        const uint64_t drain_deadline = globaltimer_ns() + 200000000ull;
        volatile int no_abort = 0;
        for (int i = 0; i < min(issued, STAGES); ++i) {
          int s = stage - 1 - i;
          uint32_t ph = phase;
          if (s < 0) {
            s += STAGES;
            ph ^= 1u;
          }
          mbar_wait(&full[s], ph, drain_deadline, &no_abort);
        }
      }
    } else if (warp == 1) {
      // ---------------- MMA issuer: one K block per TMEM buffer, alternating
      if (lane == 0) {
        int stage = 0;
        uint32_t phase = 0, it = 0;
        bool ok = true;
        for (int tile = blockIdx.x; ok && tile < num_tiles; tile += gridDim.x) {
          for (int kb = 0; kb < KB; ++kb, ++it) {
            const uint32_t buf = it & 1u;
            if (!mbar_wait(&acc_empty[buf], ((it >> 1) & 1u) ^ 1u, deadline, abort_flag) ||
                !mbar_wait(&full[stage], phase, deadline, abort_flag)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint64_t adesc = sdesc_sw128(sA + stage * A_BYTES), bdesc = sdesc_sw128(sB + stage * B_BYTES);
#pragma unroll
            for (int k = 0; k < BK / 32; ++k)
              tc_mma_f8f6f4(tmem_base + buf * BN, adesc + 2ull * k, bdesc + 2ull * k, idesc_f8f6f4(BM, BN), k != 0);
            tc_commit(&empty[stage]);
            tc_commit(&acc_full[buf]);
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
        tc_commit(mma_done);  // every MMA issued has completed before TMEM is released
        volatile int no_abort = 0;
        mbar_wait(mma_done, 0, globaltimer_ns() + 200000000ull, &no_abort);
      }
    } else if (warp == 2) {
      // ---------------- scale products, four K blocks of loads in flight
      uint32_t it = 0;
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < num_tiles; tile += gridDim.x) {
        int m_t, n_t;
        decode_tile(p, tile, m_t, n_t);
        const int nb0 = SWIGLU ? n_t : 2 * n_t, nb1 = SWIGLU ? p.NB / 2 + n_t : 2 * n_t + 1;
        const float* sa = p.sa + (int64_t)m_t * BM + 4 * lane;
        const float* sb0 = p.sb + (int64_t)nb0 * KB;
        const float* sb1 = p.sb + (int64_t)nb1 * KB;
        const bool has1 = nb1 < p.NB;
        for (int kb = 0; ok && kb < KB; kb += 4) {
          float4 a[4];
          float f0[4], f1[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (kb + j < KB) {
              a[j] = *reinterpret_cast<const float4*>(sa + (int64_t)(kb + j) * p.mp);
              f0[j] = __ldg(sb0 + kb + j);
              f1[j] = has1 ? __ldg(sb1 + kb + j) : 0.f;
            }
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (ok && kb + j < KB) {
              const uint32_t slot = it % kScaleSlots;
              ok = warp_wait(&sc_empty[slot], ((it / kScaleSlots) & 1u) ^ 1u, deadline, abort_flag);
              if (ok) {
                float4* dst = reinterpret_cast<float4*>(sF + slot * 2 * BM);
                dst[lane] = make_float4(a[j].x * f0[j], a[j].y * f0[j], a[j].z * f0[j], a[j].w * f0[j]);
                dst[32 + lane] = make_float4(a[j].x * f1[j], a[j].y * f1[j], a[j].z * f1[j], a[j].w * f1[j]);
                __syncwarp();
                if (lane == 0) mbar_arrive(&sc_full[slot]);
                ++it;
              }
            }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;\n" ::: "memory");
    // ---------------- fold and epilogue
    const int q = warp & 3;                   // TMEM lane quarter this warp may access
    const int half = (warp - EPI_BASE) >> 2;  // which half of the tile's columns
    const int row_in_tile = q * 32 + lane;
    const uint32_t t_lane = tmem_base + ((uint32_t)(q * 32) << 16);
    // this thread's two 64-column groups of the 256-column accumulator
    const int col0 = SWIGLU ? 64 * half : 128 * half;
    const int col1 = SWIGLU ? 128 + 64 * half : 128 * half + 64;
    uint32_t it = 0, tcount = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < num_tiles; tile += gridDim.x, ++tcount) {
      int m_t, n_t;
      decode_tile(p, tile, m_t, n_t);
      float acc0[64], acc1[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) acc0[i] = acc1[i] = 0.f;
      for (int kb = 0; kb < KB; ++kb, ++it) {
        const uint32_t slot = it % kScaleSlots, buf = it & 1u;
        ok = warp_wait(&sc_full[slot], (it / kScaleSlots) & 1u, deadline, abort_flag);
        if (!ok) break;
        const float f0 = sF[slot * 2 * BM + (SWIGLU ? 0 : half * BM) + row_in_tile];
        const float f1 = SWIGLU ? sF[slot * 2 * BM + BM + row_in_tile] : f0;
        ok = warp_wait(&acc_full[buf], (it >> 1) & 1u, deadline, abort_flag);
        if (!ok) break;
        if (lane == 0) mbar_arrive(&sc_empty[slot]);
        tc_fence_after();
        const uint32_t tb = t_lane + buf * BN;
        uint32_t va[32], vb[32];
        tmem_ld_32x32b_x32(tb + col0, va);
        tmem_ld_32x32b_x32(tb + col0 + 32, vb);
        tmem_wait_ld();
        fold32(acc0, va, f0);
        fold32(acc0 + 32, vb, f0);
        tmem_ld_32x32b_x32(tb + col1, va);
        tmem_ld_32x32b_x32(tb + col1 + 32, vb);
        tmem_wait_ld();
        tc_fence_before();  // this warp's reads of the buffer are complete: hand it back to the MMA warp
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[buf]);
        fold32(acc1, va, f1);
        fold32(acc1 + 32, vb, f1);
      }
      if (!ok) break;
      const int row0 = m_t * BM + q * 32;
      if constexpr (SWIGLU) {
        const int I = p.N / 2;
        const float lim = p.swiglu_limit;
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          acc0[i] = swiglu(acc0[i], acc1[i], lim);
          amax = fmaxf(amax, fabsf(acc0[i]));
        }
        // the row's other 64 h values live in the partner warp (same lane quarter, other half)
        const uint32_t par = tcount & 1u;
        s_amax[(par * 2 + half) * 128 + row_in_tile] = amax;
        mbar_arrive(&amax_bar[q * 2 + par]);
        ok = warp_wait(&amax_bar[q * 2 + par], (tcount >> 1) & 1u, deadline, abort_flag);
        if (!ok) break;
        amax = fmaxf(amax, s_amax[(par * 2 + (half ^ 1)) * 128 + row_in_tile]);
        if (row0 + lane < p.M) {
          float scale, inv;
          block_scale(amax, p.pow2, scale, inv);
          uint4* dst = reinterpret_cast<uint4*>(p.out_q + (int64_t)(row0 + lane) * I + n_t * 128 + half * 64);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float* h = acc0 + 16 * j;
            dst[j] = make_uint4(codes4(h, inv), codes4(h + 4, inv), codes4(h + 8, inv), codes4(h + 12, inv));
          }
          if (half == 0) p.out_sa[(int64_t)n_t * p.mp + row0 + lane] = scale;
        }
      } else {
        uint8_t* wb = sOut + (warp - EPI_BASE) * 2048;
        const int c0 = n_t * BN + half * 128;
        uint16_t* out0 = reinterpret_cast<uint16_t*>(p.out) + (int64_t)row0 * p.ldo + c0;
        const bool fp16 = p.out_fp16 != 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float* a = c < 2 ? acc0 + 32 * c : acc1 + 32 * (c - 2);
          uint32_t o[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = pack16(a[2 * i], a[2 * i + 1], fp16);
          store_rows(o, wb, out0 + 32 * c, p.ldo, p.M - row0, p.N - c0 - 32 * c, lane);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) report(p.status, status_word(ASAP_ST_PIPELINE_TIMEOUT, 0, 0, 16 + SWIGLU));
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

}  // namespace lin
