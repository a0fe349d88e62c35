// FP8 block-scaled linear, y = deq(xq) deq(W)^T: tiles of 128 rows x 256 weight rows on tcgen05 kind::f8f6f4.
// Included by linear.cu.
//
// y[r][n] = sum_kb sa[r][kb] * sb[n / 128][kb] * sum_{k in block kb} xq[r][k] * w[n][k].  fp32 scales are not powers
// of two and cannot ride in the MMA, so every 128-deep K block is accumulated on its own into one of two TMEM buffers
// and folded into fp32 registers (one fma per element) while the tensor core fills the other buffer.
//
// What bounds it is the turn-around of those buffers: MMA done -> a folding warp sees it -> two TMEM loads, half the
// fmas, two more loads -> the MMA issuer sees the buffer free.  A wait on an mbarrier costs about 200 cycles here even
// when its phase is long over (the MMAs keep shared memory busy), and the issuer used to make three per K block, which
// alone took 620 of its 1170 cycles.  So:
// - a K block has one barrier to start (`ready`: operands and scales landed, buffer free) and one when it is done
//   (`done`: stage free, partial complete), and both sides ask for the next one before they use the answer;
// - the activation scales come through the same ring, a K block ahead of the operands (512 bytes per block): when a block
//   is done the next one's scales have landed, and a folding warp reads them while its last fmas run;
// - a K block is issued as two halves of 128 columns, each with its own barriers and its own four folding warps: one
//   half's turn-around runs under the other's MMAs.  (Alone, MMAs of 128 columns take 710 cycles per K block, those of
//   256 take 512; folded, 950 against 1009.)
// 8192 x 8192 x 7168: 821 thousand cycles, 507 to 514 us = 1.9 PFLOP/s by itself.  In a row of launches the 1000 W cap sets
// the clock (1.65 GHz): 607 us with the quantisation's 42.
#pragma once

namespace lin {

constexpr int BM = 128, BN = 256, BK = 128;
constexpr int STAGES = 4;
constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK, B_HALF = B_BYTES / 2;
constexpr int SCALE_BYTES = BM * 4;  // a K block's activation scales
// Slots of scales: the copy for K block it + SCALE_SLOTS is issued with the operands of the block before it, after
// done(it + SCALE_SLOTS - 1 - STAGES), whose MMAs waited for every folding warp to be through with K block
// it + SCALE_SLOTS - 3 - STAGES >= it.
constexpr int SCALE_SLOTS = 8;
static_assert(SCALE_SLOTS >= STAGES + 3, "a folding warp may still read the slot");
constexpr int EPI_WARPS = 8, EPI_BASE = 4, THREADS = 32 * (EPI_BASE + EPI_WARPS);
constexpr uint32_t TMEM_COLS = 512;
constexpr int STAGE_OUT_BYTES = EPI_WARPS * 2048;
constexpr int CTRL_BYTES = 4096;  // barriers, TMEM slot, row amax exchange
constexpr int SMEM_BYTES =
    1024 + STAGES * (A_BYTES + B_BYTES) + SCALE_SLOTS * SCALE_BYTES + STAGE_OUT_BYTES + CTRL_BYTES;
static_assert(SMEM_BYTES <= 232448, "shared memory over the 227 KB per block");
// m-tiles that share a pass over the weight tiles: 16 x 9 tiles are in flight on 148 SMs, so a K block of both
// operands is read from L2 about 12 times per 128-row tile whatever M and N are.
constexpr int GROUP_M = 16;

struct Params {
  CUtensorMap tmap_a;  // activation codes [M, K], rows K padded to 128 apart
  CUtensorMap tmap_b;  // weights [N, K]
  const float* sa;     // activation scales [K blocks][mp]
  const float* sb;     // weight scales [N blocks][K blocks]
  const uint8_t* sfa;  // the same two as E8M0 atoms (linear_pow2_kernel): [mp / 128][K blocks] and
  const uint8_t* sfb;  // [K blocks][nb_atoms]
  int32_t nb_atoms;
  int64_t mp;          // M rounded up to 128
  int32_t M, N, KB, NB, m_tiles, n_tiles;
  int32_t split;       // CTAs of a cluster that share a tile's K blocks (linear only): 1, 2 or 4
  void* out;           // linear: [M, N], bf16 or fp16
  int64_t ldo;
  int32_t out_fp16;
  float swiglu_limit;  // SwiGLU: N = 2I, gate rows then up rows
  uint8_t* out_q;      // SwiGLU: codes of h [M, I]
  float* out_sa;       // SwiGLU: scales of h [I / 128][mp]
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

// A question to an mbarrier and its answer, apart: the answer stays in a predicate until it is asked for (in one statement
// a selp behind the try_wait holds the warp up for the 200 cycles that the wait is to be hidden behind).  Only of a phase
// that will end: try_wait keeps the warp for some microseconds when it does not (test_wait would not, but loses 2 to 7% of
// the product), so the last question is one whose answer is known.  ASKED declares the predicate, once in a kernel.
#define ASKED() asm volatile(".reg .pred lin_asked;")
__device__ __forceinline__ void ask(uint64_t* bar, uint32_t parity) {
  asm volatile("mbarrier.try_wait.parity.shared::cta.b64 lin_asked, [%0], %1;" ::"r"(smem_u32(bar)), "r"(parity) : "memory");
}
__device__ __forceinline__ bool answer() {
  uint32_t ok;
  asm volatile("selp.u32 %0, 1, 0, lin_asked;" : "=r"(ok)::"memory");
  return ok != 0;
}

// The same lane of a converged warp each time (the lane whose commits track its MMAs), as a predicate ptxas knows to be
// one thread's.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r));
  return r != 0;
}

// tcgen05.wait::ld that the uses of `r` cannot be moved above
__device__ __forceinline__ void tmem_wait_regs(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

// acc[2i], acc[2i + 1] += x[2i], x[2i + 1] times f: the packed fp32 fma, each half one fused multiply-add with one
// rounding.  volatile keeps them between the TMEM loads they are written between; left to the compiler's order, a K
// block took 1650 cycles instead of 900.
__device__ __forceinline__ void fold32(uint64_t* acc, const uint32_t (&x)[32], uint64_t ff) {
#pragma unroll
  for (int i = 0; i < 16; ++i)
    asm volatile("{\n\t.reg .b64 x;\n\tmov.b64 x, {%1, %2};\n\tfma.rn.f32x2 %0, x, %3, %0;\n\t}"
                 : "+l"(acc[i])
                 : "r"(x[2 * i]), "r"(x[2 * i + 1]), "l"(ff));
}
__device__ __forceinline__ uint64_t twice(float f) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(f));
  return r;
}
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(lo), "f"(hi));
  return p;
}
__device__ __forceinline__ float2 halves(uint64_t p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
  return r;
}

__device__ __forceinline__ void decode_tile(const Params& p, int tile, int& m_t, int& n_t) {
  const int per_group = GROUP_M * p.n_tiles;
  const int g = tile / per_group, local = tile - g * per_group;
  const int gm = min(GROUP_M, p.m_tiles - g * GROUP_M);
  n_t = local / gm;
  m_t = g * GROUP_M + local % gm;
}

// ---- a tile's K blocks shared by a cluster, when there are fewer tiles than SMs
// Each CTA folds its K blocks into a full tile, hands the column groups that others finish to them through shared memory
// and finishes its own: no partial goes through memory, and every sum has a fixed order.  The exchange (two barriers of
// the cluster, 128 KB written, as much or three times that read from peers) takes 4 to 5 us.  7168 x 4096 with 384 rows,
// 48 tiles, two CTAs each: 28.8 us against 38.3 unshared, E8M0 scales 24.8 against 32.7.  It is an instantiation of its
// own: in one kernel it cost the unshared tiles 8% (registers spilled in the fold).
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// A last barrier, so that no CTA leaves while another reads its shared memory; nothing is handed over, so no store has to
// be waited for.
__device__ __forceinline__ void cluster_leave() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\nbarrier.cluster.wait.aligned;\n" ::: "memory");
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
__device__ __forceinline__ float peer_load(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}
// Which of a thread's two 64-column groups (half `half` of the tile) its CTA finishes: a quarter or half of the tile each.
__device__ __forceinline__ bool finishes(int split, int rank, int half, int group) {
  return split == 1 || (split == 2 ? half == rank : half * 2 + group == rank);
}
__device__ __forceinline__ void hand_over(const uint64_t (&a)[32], float* to) {
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const float2 v = halves(a[i]);
    to[(2 * i) * 128] = v.x;
    to[(2 * i + 1) * 128] = v.y;
  }
}
__device__ __forceinline__ void take_over(uint64_t (&a)[32], const float* mine, int split, int rank) {
  for (int s = 0; s < split; ++s) {
    if (s == rank) continue;
    const uint32_t from = peer_addr(smem_u32(mine), s);
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
      float v[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = peer_load(from + (2 * i + j) * 512);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 u = halves(a[i + j]);
        a[i + j] = pair(u.x + v[2 * j], u.y + v[2 * j + 1]);
      }
    }
  }
}
// Hands the groups that other CTAs finish to them, through `part` (256 columns x 128 rows, over the operand stages), and
// adds their shares to this CTA's, in rank order.  Every warp of the cluster takes part in the barrier.
__device__ __forceinline__ void exchange(uint64_t (&a0)[32], uint64_t (&a1)[32], float* part, int split, int rank, int half,
                                         int row, bool ok) {
  static_assert(BM * BN * 4 <= STAGES * (A_BYTES + B_BYTES), "the partials lie over the operand stages");
  float* mine = part + half * 128 * 128 + row;
  if (ok && !finishes(split, rank, half, 0)) hand_over(a0, mine);
  if (ok && !finishes(split, rank, half, 1)) hand_over(a1, mine + 64 * 128);
  __syncwarp();
  cluster_sync();
  if (ok && finishes(split, rank, half, 0)) take_over(a0, mine, split, rank);
  if (ok && finishes(split, rank, half, 1)) take_over(a1, mine + 64 * 128, split, rank);
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
template <int SWIGLU, bool SPLIT = false>
__global__ void __launch_bounds__(THREADS, 1) linear_gemm_kernel(const __grid_constant__ Params p) {
  ASKED();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + STAGES * A_BYTES;
  float* sSa = reinterpret_cast<float*>(sB + STAGES * B_BYTES);  // [SCALE_SLOTS][BM]
  uint8_t* sOut = reinterpret_cast<uint8_t*>(sSa) + SCALE_SLOTS * SCALE_BYTES;
  uint8_t* ctrl = sOut + STAGE_OUT_BYTES;
  // K block `it` uses stage it % STAGES, scale slot it % SCALE_SLOTS and TMEM buffer it % 2
  uint64_t* ready = reinterpret_cast<uint64_t*>(ctrl);  // [STAGES][2 halves] operands, scales, buffer: the MMAs may start
  uint64_t* done = ready + 2 * STAGES;                  // [STAGES][2] the half's MMAs have completed
  uint64_t* mma_done = done + 2 * STAGES;
  uint64_t* amax_bar = mma_done + 1;  // [4 lane quarters][2 tile parities]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ctrl + 512);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(ctrl + 516);
  float* s_amax = reinterpret_cast<float*>(ctrl + 1024);  // [2 tile parities][2 halves][128 rows]

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2 * STAGES; ++s) {
      mbar_init(&ready[s], 1 + EPI_WARPS / 2);
      mbar_init(&done[s], 1);
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
  const int num_tiles = p.m_tiles * p.n_tiles;
  // with split > 1 a cluster has one tile, and this CTA the K blocks [kb0, kb0 + KB) of it
  const int split = SPLIT ? p.split : 1, rank = SPLIT ? (int)cluster_rank() : 0;
  const int kb0 = rank * p.KB / split, KB = (rank + 1) * p.KB / split - kb0;
  const int tile0 = blockIdx.x / split, tile_step = gridDim.x / split;
  const uint64_t deadline = globaltimer_ns() + p.timeout_ns;

  // Registers (as launched 384 x 168 = 64512): the four helper warps give theirs up (two idle), the folding warps hold the
  // 128 accumulators and two TMEM loads in flight: 128 x 64 + 256 x 216 = 63488.
  if (warp < EPI_BASE) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;\n" ::: "memory");
    if (warp == 0) {
      // ---------------- TMA producer
      if (lane == 0) {
        int stage = 0;
        uint32_t phase = 0, it = 0;
        bool ok = true;
        for (int tile = tile0; ok && tile < num_tiles; tile += tile_step) {
          int m_t, n_t;
          decode_tile(p, tile, m_t, n_t);
          const float* sa = p.sa + (int64_t)m_t * BM + kb0 * p.mp;
          const int b0 = SWIGLU ? n_t * 128 : n_t * BN, b1 = SWIGLU ? p.N / 2 + n_t * 128 : n_t * BN + 128;
          for (int kb = 0; kb < KB; ++kb, ++it) {
            // (the second half's commit follows the first's, so it speaks for both)
            if (!mbar_wait(&done[2 * stage + 1], phase ^ 1u, deadline, abort_flag)) {
              ok = false;
              break;
            }
            const int scales = (kb == 0) + (kb + 1 < KB);
            uint64_t* bar = &ready[2 * stage];
            uint8_t* b = sB + stage * B_BYTES;
            mbar_arrive_expect_tx(bar, A_BYTES + B_HALF + scales * SCALE_BYTES);
            tma_load_2d(sA + stage * A_BYTES, &p.tmap_a, (kb0 + kb) * BK, m_t * BM, bar);
            if (kb == 0) bulk_load(sSa + it % SCALE_SLOTS * BM, sa, SCALE_BYTES, bar);
            if (kb + 1 < KB)
              bulk_load(sSa + (it + 1) % SCALE_SLOTS * BM, sa + (int64_t)(kb + 1) * p.mp, SCALE_BYTES, bar);
            if constexpr (SWIGLU) {  // boxes of 64 rows: a half holds 64 gate rows and the 64 up rows they meet
              tma_load_2d(b, &p.tmap_b, (kb0 + kb) * BK, b0, bar);
              tma_load_2d(b + B_HALF / 2, &p.tmap_b, (kb0 + kb) * BK, b1, bar);
              mbar_arrive_expect_tx(bar + 1, B_HALF);
              tma_load_2d(b + B_HALF, &p.tmap_b, (kb0 + kb) * BK, b0 + 64, bar + 1);
              tma_load_2d(b + B_HALF + B_HALF / 2, &p.tmap_b, (kb0 + kb) * BK, b1 + 64, bar + 1);
            } else {
              tma_load_2d(b, &p.tmap_b, (kb0 + kb) * BK, b0, bar);
              mbar_arrive_expect_tx(bar + 1, B_HALF);
              tma_load_2d(b + B_HALF, &p.tmap_b, (kb0 + kb) * BK, b1, bar + 1);
            }
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
      }
    } else if (warp == 1) {
      // ---------------- MMA issuer: one K block per TMEM buffer, alternating.  The warp runs the loop as a whole and one
      // elected lane issues, so that descriptors stay in uniform registers (5% of a K block's time).
      {
        // Halves are numbered through: half x is K block x / 2, barrier pair x % (2 STAGES).  Whether the next half may
        // start is asked before this half's MMAs are issued, and the answer used after.
        const uint32_t total = (uint32_t)((num_tiles - tile0 + tile_step - 1) / tile_step) * (uint32_t)KB * 2u;
        bool ok = true, early = false;
        for (uint32_t x = 0; ok && x < total; ++x) {
          const uint32_t slot = x % (2 * STAGES), stage = slot / 2, h = x & 1u, next = x + 1 < total ? x + 1 : x;
          const uint64_t adesc = sdesc_sw128(sA + stage * A_BYTES);
          const uint64_t bdesc = sdesc_sw128(sB + stage * B_BYTES + h * B_HALF);
          const uint32_t acc = tmem_base + ((x >> 1) & 1u) * BN + h * 128;
          if (!early) ok = __all_sync(0xffffffffu, mbar_wait(&ready[slot], (x / (2 * STAGES)) & 1u, deadline, abort_flag));
          if (!ok) break;
          ask(&ready[next % (2 * STAGES)], (next / (2 * STAGES)) & 1u);
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < BK / 32; ++k)
              tc_mma_f8f6f4(acc, adesc + 2ull * k, bdesc + 2ull * k, idesc_f8f6f4(BM, 128), k != 0);
            tc_commit(&done[slot]);
          }
          early = __all_sync(0xffffffffu, answer());
        }
        __syncwarp();
        if (elect_one()) tc_commit(mma_done);
        __syncwarp();
        drain_mmas(mma_done, deadline, abort_flag);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;\n" ::: "memory");
    // ---------------- fold and epilogue
    const int q = warp & 3;                   // TMEM lane quarter this warp may access
    const int half = (warp - EPI_BASE) >> 2;  // which half of the tile's columns
    const int row_in_tile = q * 32 + lane;
    const uint32_t t_lane = tmem_base + ((uint32_t)(q * 32) << 16);
    // this thread's two 64-column groups of the 256-column accumulator (SwiGLU: gate, then the up they meet)
    const int col0 = 128 * half, col1 = 128 * half + 64;
    uint32_t it = 0, tcount = 0;
    bool ok = true, exchanged = false;
    if (lane == 0) {  // both TMEM buffers start free
      mbar_arrive(&ready[half]);
      mbar_arrive(&ready[2 + half]);
    }
    for (int tile = tile0; ok && tile < num_tiles; tile += tile_step, ++tcount) {
      int m_t, n_t;
      decode_tile(p, tile, m_t, n_t);
      // the weight blocks of the two column groups (a block behind the last has no columns that are stored)
      const int nb = SWIGLU ? n_t : min(2 * n_t + half, p.NB - 1);
      const float* sb0 = p.sb + (int64_t)nb * p.KB + kb0;
      const float* sb1 = p.sb + (int64_t)(p.NB / 2 + nb) * p.KB;  // SwiGLU only
      float b0 = __ldg(sb0), b1 = SWIGLU ? __ldg(sb1) : 0.f;
      uint64_t acc0[32], acc1[32];  // pairs of columns
#pragma unroll
      for (int i = 0; i < 32; ++i) acc0[i] = acc1[i] = 0;
      // 64 columns are loaded while the 64 before them are folded, across K blocks as well
      uint32_t va[32], vb[32];
      ok = warp_wait(&done[2 * (it % STAGES) + half], (it / STAGES) & 1u, abort_flag);
      if (!ok) break;
      tc_fence_after();
      tmem_ld_32x32b_x32(t_lane + (it & 1u) * BN + col0, va);
      tmem_ld_32x32b_x32(t_lane + (it & 1u) * BN + col0 + 32, vb);
      float sa = sSa[it % SCALE_SLOTS * BM + row_in_tile];
      for (int kb = 0; kb < KB; ++kb, ++it) {
        const uint32_t tb = t_lane + (it & 1u) * BN;
        const bool more = kb + 1 < KB;
        const uint64_t f0 = twice(sa * b0), f1 = SWIGLU ? twice(sa * b1) : f0;
        if (more) {  // the next block's factors; its scales landed before this block's MMAs started
          sa = sSa[(it + 1) % SCALE_SLOTS * BM + row_in_tile];
          b0 = __ldg(sb0 + kb + 1);
          if (SWIGLU) b1 = __ldg(sb1 + kb + 1);
        }
        tmem_wait_regs(va);
        tmem_wait_regs(vb);
        fold32(acc0, va, f0);
        tmem_ld_32x32b_x32(tb + col1, va);
        fold32(acc0 + 16, vb, f0);
        tmem_ld_32x32b_x32(tb + col1 + 32, vb);
        // asked early: by the time the answer is used the next block is usually done
        const uint32_t next = it + more;
        ask(&done[2 * (next % STAGES) + half], (next / STAGES) & 1u);
        tmem_wait_regs(va);
        tmem_wait_regs(vb);
        tc_fence_before();  // this warp's reads of the buffer are complete: K block it + 2 may have it
        __syncwarp();
        if (lane == 0) mbar_arrive(&ready[2 * ((it + 2) % STAGES) + half]);
        if (!__all_sync(0xffffffffu, answer()) && more) {
          ok = warp_wait(&done[2 * ((it + 1) % STAGES) + half], ((it + 1) / STAGES) & 1u, abort_flag);
          if (!ok) break;
        }
        tc_fence_after();
        const uint32_t tn = t_lane + ((it + 1) & 1u) * BN;
        fold32(acc1, va, f1);
        if (more) tmem_ld_32x32b_x32(tn + col0, va);
        fold32(acc1 + 16, vb, f1);
        if (more) tmem_ld_32x32b_x32(tn + col0 + 32, vb);
      }
      if (!ok) break;
      const int row0 = m_t * BM + q * 32;
      if constexpr (SWIGLU) {
        const int I = p.N / 2;
        const float lim = p.swiglu_limit;
        float amax = 0.f, h[64];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float2 g = halves(acc0[i]), u = halves(acc1[i]);
          h[2 * i] = swiglu(g.x, u.x, lim);
          h[2 * i + 1] = swiglu(g.y, u.y, lim);
          amax = fmaxf(amax, fmaxf(fabsf(h[2 * i]), fabsf(h[2 * i + 1])));
        }
        // the row's other 64 h values live in the partner warp (same lane quarter, other half)
        const uint32_t par = tcount & 1u;
        s_amax[(par * 2 + half) * 128 + row_in_tile] = amax;
        mbar_arrive(&amax_bar[q * 2 + par]);
        ok = warp_wait(&amax_bar[q * 2 + par], (tcount >> 1) & 1u, abort_flag);
        if (!ok) break;
        amax = fmaxf(amax, s_amax[(par * 2 + (half ^ 1)) * 128 + row_in_tile]);
        if (row0 + lane < p.M) {
          float scale, inv;
          block_scale(amax, false, scale, inv);
          uint4* dst = reinterpret_cast<uint4*>(p.out_q + (int64_t)(row0 + lane) * I + n_t * 128 + half * 64);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            dst[j] = make_uint4(codes4(h + 16 * j, inv), codes4(h + 16 * j + 4, inv), codes4(h + 16 * j + 8, inv),
                                codes4(h + 16 * j + 12, inv));
          if (half == 0) p.out_sa[(int64_t)n_t * p.mp + row0 + lane] = scale;
        }
      } else {
        uint8_t* wb = sOut + (warp - EPI_BASE) * 2048;
        const int c0 = n_t * BN + half * 128;
        uint16_t* out0 = reinterpret_cast<uint16_t*>(p.out) + (int64_t)row0 * p.ldo + c0;
        const bool fp16 = p.out_fp16 != 0;
        if constexpr (SPLIT) {
          // the partials take the place of the operands: both halves' MMAs have to be done with those
          ok = warp_wait(&done[2 * ((it - 1) % STAGES) + 1], ((it - 1) / STAGES) & 1u, abort_flag);
          exchange(acc0, acc1, reinterpret_cast<float*>(sA), split, rank, half, row_in_tile, ok);
          exchanged = true;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (SPLIT && (!ok || !finishes(split, rank, half, c / 2))) continue;
          const uint64_t* a = c < 2 ? acc0 + 16 * c : acc1 + 16 * (c - 2);
          uint32_t o[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 v = halves(a[i]);
            o[i] = pack16(v.x, v.y, fp16);
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
    if (warp < EPI_BASE) cluster_sync();  // the exchange's barrier
    cluster_leave();
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {  // copies may still be on their way into this block's shared memory: let them land before it ends
    if (threadIdx.x == 0) report(p.status, status_word(ASAP_ST_PIPELINE_TIMEOUT, 0, 0, 16 + SWIGLU));
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
