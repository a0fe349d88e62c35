// libasap dense side of the MoE layer: the FP8 block-scaled linear and the FP8 shared expert of an attention rank
// (the checkpoint's E4M3 weights with one scale per 128 x 128 block, the format asap_experts_register_fp8 takes for
// the routed experts).  The reference leaves the shared expert to SGLang's linear layers
// (python/sgl_asap_plugin/srt/batch_overlap/operations_strategy.py:106-111 adds its output to the routed one).
#include <cuda.h>
#include <cuda_fp16.h>
#include <string.h>

#include <mutex>
#include <new>
#include <unordered_map>

#include "common.cuh"
#include "tmap.cuh"
#include "waits.cuh"

namespace asap {

int sm_count();

namespace lin {

constexpr float kE4M3Max = 448.f;
constexpr int kMaxSmem = 232448;  // shared memory a block may have

// Scale of one block of activations and the factor that maps it to the code range.  The absolute maximum counts as at
// least 1e-10, so a block of zeros has codes 0.  pow2: amax / 448 rounded up to a power of two, by its bits (448 =
// 1.75 * 2^8); an infinite block gets NaN codes, which is what inf * (448 / inf) gives the other form.
__device__ __forceinline__ void block_scale(float amax, bool pow2, float& scale, float& inv) {
  const float a = fmaxf(amax, 1e-10f);
  if (!pow2) {
    scale = a / kE4M3Max;
    inv = kE4M3Max / a;
    return;
  }
  const uint32_t bits = __float_as_uint(a);
  const uint32_t e = (bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u);
  scale = __uint_as_float(e << 23);
  inv = (bits >> 23) == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float((254 - e) << 23);
}

// E4M3 codes of 4 values, round to nearest even, saturating; NaN stays NaN
__device__ __forceinline__ uint32_t codes4(const float* v, float inv) {
  return cvt_e4m3x2(v[0] * inv, v[1] * inv) | (cvt_e4m3x2(v[2] * inv, v[3] * inv) << 16);
}

// A half-warp's block of 128 16-bit values, 8 per lane -> this lane's 8 codes, and the block's scale
__device__ __forceinline__ void quant8(const uint4& u, bool fp16, bool pow2, uint2& codes, float& scale) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  float v[8], amax = 0.f, inv;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = fp16 ? __half22float2(*reinterpret_cast<const __half2*>(&w[j]))
                          : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[j]));
    v[2 * j] = f.x;
    v[2 * j + 1] = f.y;
    amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  block_scale(amax, pow2, scale, inv);
  codes = make_uint2(codes4(v, inv), codes4(v + 4, inv));
}

// fminf and fmaxf would give the limit for a NaN; these give the NaN.  (So do two comparisons, but they spill in the fold
// kernel: 2% of a shared expert of 16384 tokens.)
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float swiglu(float g, float u, float limit) {
  if (limit > 0.f) {
    g = min_nan(g, limit);
    u = min_nan(max_nan(u, -limit), limit);
  }
  return __fdividef(g, 1.f + expf(-g)) * u;  // within 2 ulp; a denominator above 2^126 gives 0, the value to 10^-36
}

}  // namespace lin

#include "gemm_linear.cuh"
#include "gemm_pow2.cuh"
#include "gemm_skinny.cuh"

namespace lin {

// ------------------------------------------------------------------ activation quantisation
// x [M, K] -> codes [M, 128 * KB] (K padded with 0) and scales: fp32 [KB][mp], or E8M0 atoms when they are powers of
// two.  A half-warp holds a block, 8 values per lane.  Bound by memory; a warp has QUANT_AHEAD loads of 512 bytes in
// flight before it uses the first.
struct QuantArgs {
  const uint16_t* x;
  int64_t ldx;
  int32_t M, K, KB, fp16, pow2, atoms;
  int64_t mp;
  uint8_t* xq;
  float* sa;
};

constexpr int QUANT_AHEAD = 4;
__global__ void __launch_bounds__(256) quant_rows_kernel(const __grid_constant__ QuantArgs p) {
  const int lane = threadIdx.x & 31;
  const uint32_t groups = (p.KB + 2 * QUANT_AHEAD - 1) / (2 * QUANT_AHEAD);  // of QUANT_AHEAD x 256 values
  const uint32_t items = p.M * groups, step = gridDim.x * (blockDim.x >> 5);
  grid_dependents_launch();
  for (uint32_t i = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); i < items; i += step) {
    const uint32_t row = i / groups;
    const int col0 = (int)(i - row * groups) * QUANT_AHEAD * 256 + lane * 8;
    const uint16_t* x = p.x + (int64_t)row * p.ldx;
    uint4 u[QUANT_AHEAD];
#pragma unroll
    for (int j = 0; j < QUANT_AHEAD; ++j) {
      const int col = col0 + 256 * j;
      u[j] = make_uint4(0, 0, 0, 0);
      if (col < p.K) u[j] = *reinterpret_cast<const uint4*>(x + col);
    }
#pragma unroll
    for (int j = 0; j < QUANT_AHEAD; ++j) {
      const int col = col0 + 256 * j;
      if (col - lane * 8 >= p.KB * 128) break;
      uint2 codes;
      float scale;
      quant8(u[j], p.fp16 != 0, p.pow2 != 0, codes, scale);
      if (col < p.KB * 128) {
        *reinterpret_cast<uint2*>(p.xq + (int64_t)row * p.KB * 128 + col) = codes;
        if ((lane & 15) == 0) {
          const int kb = col / 128;
          if (p.atoms)
            *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(p.sa) + atom_off(row, kb, p.KB)) = atom_word(scale);
          else p.sa[(int64_t)kb * p.mp + row] = scale;
        }
      }
    }
  }
}

// ------------------------------------------------------------------ host side
struct Linear {
  asap_fp8_linear_t d;
  CUtensorMap map;
  int32_t KB, NB;
};

static std::mutex g_mu;
static std::unordered_map<uint64_t, Linear*> g_linear;
static uint64_t g_next = 1;

static Linear* find(uint64_t h) {
  std::lock_guard<std::mutex> lk(g_mu);
  auto it = g_linear.find(h);
  return it == g_linear.end() ? nullptr : it->second;
}

static int ensure_attrs() {
  static std::mutex mu;
  static bool done[64] = {};
  int dev = 0;
  ASAP_CUDA(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> lk(mu);
  if (dev >= 0 && dev < 64 && done[dev]) return ASAP_OK;
  ASAP_CUDA(cudaFuncSetAttribute(linear_gemm_kernel<0>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
  ASAP_CUDA(cudaFuncSetAttribute(linear_gemm_kernel<0, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
  ASAP_CUDA(cudaFuncSetAttribute(linear_gemm_kernel<1>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
  ASAP_CUDA(cudaFuncSetAttribute(linear_pow2_kernel<0>, cudaFuncAttributeMaxDynamicSharedMemorySize, P2_SMEM_BYTES));
  ASAP_CUDA(
      cudaFuncSetAttribute(linear_pow2_kernel<0, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, P2_SMEM_BYTES));
  ASAP_CUDA(cudaFuncSetAttribute(linear_pow2_kernel<1>, cudaFuncAttributeMaxDynamicSharedMemorySize, P2_SMEM_BYTES));
  for (const void* f : {(const void*)linear_skinny_kernel<16, 0, 0>, (const void*)linear_skinny_kernel<16, 0, 1>,
                        (const void*)linear_skinny_kernel<32, 0, 1>, (const void*)linear_skinny_kernel<64, 0, 1>,
                        (const void*)linear_skinny_kernel<128, 0, 1>, (const void*)linear_skinny_kernel<16, 1, 1>,
                        (const void*)linear_skinny_kernel<32, 1, 1>, (const void*)linear_skinny_kernel<64, 1, 1>}) {
    ASAP_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem));
    ASAP_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
  }
  if (dev >= 0 && dev < 64) done[dev] = true;
  return ASAP_OK;
}

// Workspace of one product's activations: codes, then scales.
struct ActWs {
  int64_t mp;
  uint64_t codes, scales;  // bytes
};
static ActWs act_ws(int64_t m, int64_t k) {
  const uint64_t kb = (k + 127) / 128;
  ActWs w;
  w.mp = (m + 127) / 128 * 128;
  w.codes = align_up((uint64_t)m * kb * 128, 256);
  w.scales = align_up(kb * w.mp * 4, 256);
  return w;
}

static int check_rows(const char* fn, int32_t m, uint64_t x, int64_t ldx, int32_t k, uint64_t out, uint64_t ws,
                      uint64_t have, uint64_t need) {
  if (m < 1 || m > ASAP_LINEAR_MAX_ROWS) {
    set_error("%s: %d rows, need 1 to %d", fn, m, ASAP_LINEAR_MAX_ROWS);
    return ASAP_EINVAL;
  }
  if (!x || (x & 15) || ldx < k || (ldx & 7)) {
    set_error("%s: x must be 16-byte aligned with a row stride of at least %d and a multiple of 8 (got %lld)", fn, k,
              (long long)ldx);
    return ASAP_EINVAL;
  }
  if (!out || (out & 15) || (need && (!ws || (ws & 255) || have < need))) {
    set_error("%s: out must be 16-byte and the workspace 256-byte aligned and hold %llu bytes (got %llu)", fn,
              (unsigned long long)need, (unsigned long long)have);
    return ASAP_EINVAL;
  }
  return ASAP_OK;
}

static int quantise(uint64_t x, int64_t ldx, int32_t m, const Linear* L, int32_t fp16, bool atoms, uint64_t xq,
                    uint64_t sa, int64_t mp, cudaStream_t st) {
  QuantArgs q{};
  q.x = (const uint16_t*)x;
  q.ldx = ldx;
  q.M = m;
  q.K = L->d.k;
  q.KB = L->KB;
  q.fp16 = fp16;
  q.pow2 = L->d.atoms != 0;
  q.atoms = atoms;
  q.mp = mp;
  q.xq = (uint8_t*)xq;
  q.sa = (float*)sa;
  const int64_t items = (int64_t)m * ((L->KB + 2 * QUANT_AHEAD - 1) / (2 * QUANT_AHEAD));
  const int64_t blocks = (items + 7) / 8, cap = 8ll * sm_count();
  quant_rows_kernel<<<(int)(blocks < cap ? blocks : cap), 256, 0, st>>>(q);
  ASAP_CHECK_LAUNCH("quant_rows_kernel");
  return ASAP_OK;
}

static int tile_split(const Linear* L, bool swiglu, int32_t m);

// One product over quantised activations.  swiglu: L holds gate rows then up rows, h goes to out_q / out_sa.
static int product(const Linear* L, bool swiglu, uint64_t xq, uint64_t sa, int32_t m, int64_t mp, uint64_t out,
                   int64_t ldo, int32_t fp16, float limit, uint64_t out_q, uint64_t out_sa, uint64_t status,
                   uint64_t timeout_ns, cudaStream_t st) {
  Params p;
  memset(&p, 0, sizeof(p));
  if (int rc = make_tmap_2d(&p.tmap_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, (const void*)xq, (uint64_t)L->KB * 128, m,
                            (uint64_t)L->KB * 128, BK, BM, "activation codes"))
    return rc;
  p.tmap_b = L->map;
  if (swiglu && !L->d.atoms)  // boxes of 64 rows
    if (int rc = make_tmap_2d(&p.tmap_b, CU_TENSOR_MAP_DATA_TYPE_UINT8, (const void*)L->d.w, L->d.k, L->d.n, L->d.k, BK, 64,
                              "gate and up weights"))
      return rc;
  p.sa = (const float*)sa;
  p.sb = (const float*)L->d.scale;
  p.sfa = (const uint8_t*)sa;
  p.sfb = (const uint8_t*)L->d.atoms;
  p.nb_atoms = (L->NB + 1) / 2 * 2;
  p.mp = mp;
  p.M = m;
  p.N = L->d.n;
  p.KB = L->KB;
  p.NB = L->NB;
  p.m_tiles = (m + BM - 1) / BM;
  p.n_tiles = swiglu ? L->d.n / 256 : (L->d.n + BN - 1) / BN;
  p.out = (void*)out;
  p.ldo = ldo;
  p.out_fp16 = fp16;
  p.swiglu_limit = limit;
  p.out_q = (uint8_t*)out_q;
  p.out_sa = (float*)out_sa;
  p.status = status;
  p.timeout_ns = timeout_ns;
  p.split = tile_split(L, swiglu, m);
  const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.split > 1 ? tiles * p.split : tiles < sm_count() ? tiles : sm_count()));
  cfg.blockDim = dim3(L->d.atoms ? P2_THREADS : THREADS);
  cfg.dynamicSmemBytes = L->d.atoms ? P2_SMEM_BYTES : SMEM_BYTES;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = p.split;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = p.split > 1 ? 1 : 0;
  void (*kernel)(Params) = L->d.atoms ? (swiglu ? linear_pow2_kernel<1> : linear_pow2_kernel<0>)
                                      : (swiglu ? linear_gemm_kernel<1> : linear_gemm_kernel<0>);
  if (p.split > 1) kernel = L->d.atoms ? linear_pow2_kernel<0, true> : linear_gemm_kernel<0, true>;
  ASAP_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
  return ASAP_OK;
}

// ------------------------------------------------------------------ few rows
// Up to here the few-rows linear quantises its rows itself.  7168 x 4096: 1 row 10.8 us against 11.0 with a kernel before
// it (2064 x 1040: 5.3 against 5.8), and one launch less for the caller; 8 rows 13.1 against 11.7.  Only the linear: the
// shared expert's rows come quantised from the first one on, as its second product's do.
constexpr int kInKernelRows = 4;
constexpr int kInKernelDim = SK_MAX_KB * SK_MAX_SPLIT * BK;  // and this many values of K, whose codes fit the clusters

// How a product of few rows is launched.  rounds: K blocks that a CTA works through, times the waves of clusters.
struct SkinnyPlan {
  int tmpl, tn, split, stages, max_kb, smem;
  int64_t rounds;
  explicit operator bool() const { return split > 0; }
};

// Clusters of `split` CTAs that run at once, with two CTAs (half an SM's shared memory) or one on an SM.  A cluster lies
// within one GPC, so eight to a cluster leave SMs idle that two would use.
static int clusters_at_once(int split, bool two) {
  static std::mutex mu;
  static int cached[64][4] = {};
  int dev = 0, log = split == 1 ? 0 : split == 2 ? 1 : split == 4 ? 2 : 3;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  std::lock_guard<std::mutex> lk(mu);
  int& n = cached[dev][log];
  if (!n) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(split * 1024);
    cfg.blockDim = dim3(SK_THREADS);
    cfg.dynamicSmemBytes = kMaxSmem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = split;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, linear_skinny_kernel<16, 0, 0>, &cfg) != cudaSuccess || n < 1) {
      (void)cudaGetLastError();
      n = sm_count() / split;
    }
  }
  return two ? 2 * n : n;  // the query knows nothing of two: it answers one CTA to an SM for whatever uses tensor memory
}

// The rows are cut into equal column tiles of the MMA, of at most 128 (64 with SwiGLU, whose weight tiles are two), and
// the kernel is compiled for 16, 32, 64 and 128.  K is split as far as all clusters still run at once: with two CTAs on an
// SM where a folding warp holds at most 32 columns and three stages fit half an SM's shared memory, else one.
template <int SWIGLU, int XTMA>
static SkinnyPlan skinny_plan(const Linear* L, int32_t m) {
  const int n_tiles = SWIGLU ? L->d.n / 256 : (L->d.n + 127) / 128;
  for (int cap = XTMA ? (SWIGLU ? 64 : 128) : 16; cap >= 16; cap /= 2) {
    const int64_t y = (m + cap - 1) / cap;
    if (y > 65535) continue;
    SkinnyPlan pl{};
    pl.tn = ((int)((m + y - 1) / y) + 15) / 16 * 16;
    pl.tmpl = pl.tn <= 16 ? 16 : pl.tn <= 32 ? 32 : pl.tn <= 64 ? 64 : 128;
    const int tiles = SWIGLU ? 2 : 1;
    const int stage = tiles * 128 * BK + (XTMA ? pl.tmpl * BK : 0), part = tiles * pl.tmpl * 512;
    const int least = part > 3 * stage ? (part + stage - 1) / stage : 3;
    const int half = kMaxSmem / 2 - 1024;
    auto fixed = [&](int split) {
      return 1024 + 2048 + (L->KB + split - 1) / split * ((XTMA ? 0 : pl.tmpl * BK) + pl.tmpl * 4 + 8);
    };
    auto two = [&](int split) { return tiles * pl.tmpl <= 64 && fixed(split) + least * stage <= half; };
    auto fits = [&](int split) {
      return (L->KB + split - 1) / split <= SK_MAX_KB && fixed(split) + least * stage <= kMaxSmem;
    };
    pl.split = 1;
    while (2 * pl.split <= SK_MAX_SPLIT && 2 * pl.split <= L->KB &&
           (!fits(pl.split) || n_tiles * y <= clusters_at_once(2 * pl.split, two(2 * pl.split))))
      pl.split *= 2;
    if (!fits(pl.split)) continue;
    const int at_once = clusters_at_once(pl.split, two(pl.split));
    pl.max_kb = (L->KB + pl.split - 1) / pl.split;
    pl.rounds = (n_tiles * y + at_once - 1) / at_once * pl.max_kb;
    pl.stages = ((two(pl.split) ? half : kMaxSmem) - fixed(pl.split)) / stage;
    if (pl.stages > SK_MAX_STAGES) pl.stages = SK_MAX_STAGES;
    if (pl.stages > pl.max_kb) pl.stages = pl.max_kb;
    if (pl.stages < least) pl.stages = least;
    pl.smem = fixed(pl.split) + pl.stages * stage;
    // Never more CTAs on an SM than its tensor memory holds, of one launch or of two on different streams: a CTA that
    // waits for tensor memory holds up its cluster, which may hold what another one waits for.  Two with 256 columns
    // (80 KB: a third does not fit the SM's 228 KB), one with 512 (150 KB: not beside one of 80 either).
    const int alone = (tiles * pl.tmpl <= 64 ? 80 : 150) * 1024;
    if (pl.smem < alone) pl.smem = alone;
    return pl;
  }
  return SkinnyPlan{};
}

// The product in 128 x 256 tiles: the CTAs of a cluster that share a tile's K blocks, where there are fewer tiles than SMs
// and the K blocks saved are worth the exchange of the partials.  That takes 4 to 5 us, 10 K blocks' time: 7168 x 4096 with
// 384 rows saves 28 blocks and 9.5 us; 2048 x 7168 with 160 rows (16 blocks) is the same shared or not, 17.5 us.  SwiGLU
// needs a row's whole 128 h in one CTA and does not share.
constexpr int kExchange = 10;
static int64_t tile_rounds(const Linear* L, bool swiglu, int32_t m, int split) {
  const int64_t tiles = (int64_t)((m + BM - 1) / BM) * (swiglu ? L->d.n / 256 : (L->d.n + BN - 1) / BN);
  if (split > 1 && (swiglu || split > L->KB || tiles > clusters_at_once(split, false))) return INT64_MAX;
  if (split > 1) return (L->KB + split - 1) / split + kExchange;
  return (tiles + sm_count() - 1) / sm_count() * L->KB;
}
static int tile_split(const Linear* L, bool swiglu, int32_t m) {
  int best = 1;
  for (int s = 2; s <= 4; s *= 2)
    if (tile_rounds(L, swiglu, m, s) < tile_rounds(L, swiglu, m, best)) best = s;
  return best;
}
// The measure that chooses between tiles and few rows: a K block takes either kernel 0.4 to 0.7 us, so the one with fewer
// rounds is taken.  7168 x 4096 with 256 rows: 24 rounds in shared tiles 25.4 us, 28 of the few-rows form 27.1, 56 in
// tiles of one CTA 39.4.
static int64_t tile_rounds(const Linear* L, bool swiglu, int32_t m) {
  return tile_rounds(L, swiglu, m, tile_split(L, swiglu, m));
}

// What is the same for every launch of a call
static SkinnyParams skinny_params(uint64_t x, int64_t ldx, int32_t m, int32_t fp16, int64_t mp, uint64_t status,
                                  uint64_t timeout_ns) {
  SkinnyParams p;
  memset(&p, 0, sizeof(p));
  p.x = (const uint16_t*)x;
  p.ldx = ldx;
  p.M = m;
  p.fp16 = fp16;
  p.mp = mp;
  p.status = status;
  p.timeout_ns = timeout_ns;
  return p;
}

// xq / sa: the quantised rows (XTMA), from a kernel launched just before on the same stream
template <int SWIGLU, int XTMA>
static int skinny(const Linear* L, const SkinnyPlan& pl, SkinnyParams& p, uint64_t xq, uint64_t sa, cudaStream_t st) {
  p.tmap_w = L->map;
  if (XTMA)
    if (int rc = make_tmap_2d(&p.tmap_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, (const void*)xq, (uint64_t)L->KB * 128, p.M,
                              (uint64_t)L->KB * 128, BK, pl.tn, "activation codes"))
      return rc;
  p.sa = (const float*)sa;
  p.K = L->d.k;
  p.N = L->d.n;
  p.KB = L->KB;
  p.NB = L->NB;
  p.split = pl.split;
  p.stages = pl.stages;
  p.max_kb = pl.max_kb;
  p.tn = pl.tn;
  p.sb = (const float*)L->d.scale;
  p.pow2 = L->d.atoms != 0;
  const int n_tiles = SWIGLU ? L->d.n / 256 : (L->d.n + 127) / 128;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(n_tiles * pl.split, (p.M + pl.tn - 1) / pl.tn);
  cfg.blockDim = dim3(SK_THREADS);
  cfg.dynamicSmemBytes = pl.smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = pl.split;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = XTMA ? 2 : 1;
  if (pl.tmpl == 16) ASAP_CUDA(cudaLaunchKernelEx(&cfg, linear_skinny_kernel<16, SWIGLU, XTMA>, p));
  else if constexpr (XTMA) {
    if (pl.tmpl == 32) ASAP_CUDA(cudaLaunchKernelEx(&cfg, linear_skinny_kernel<32, SWIGLU, 1>, p));
    else if (pl.tmpl == 64) ASAP_CUDA(cudaLaunchKernelEx(&cfg, linear_skinny_kernel<64, SWIGLU, 1>, p));
    else if constexpr (!SWIGLU) ASAP_CUDA(cudaLaunchKernelEx(&cfg, linear_skinny_kernel<128, 0, 1>, p));
  }
  return ASAP_OK;
}

}  // namespace lin
}  // namespace asap

using namespace asap;

extern "C" {

int asap_fp8_linear_register(const asap_fp8_linear_t* d, uint64_t* handle) {
  if (!d || !handle) {
    set_error("asap_fp8_linear_register: NULL argument");
    return ASAP_EINVAL;
  }
  if (d->n < 16 || d->k < 16 || d->n % 16 || d->k % 16 || d->n > ASAP_LINEAR_MAX_DIM || d->k > ASAP_LINEAR_MAX_DIM) {
    set_error("asap_fp8_linear_register: n and k must be multiples of 16 from 16 to %d (got %d, %d)",
              ASAP_LINEAR_MAX_DIM, d->n, d->k);
    return ASAP_EINVAL;
  }
  if (!d->w || (d->w & 15) || !d->scale || (d->scale & 3) || (d->atoms & 15)) {
    set_error("asap_fp8_linear_register: weights must be 16-byte and scales 4-byte aligned, non-NULL, atoms 16-byte");
    return ASAP_EINVAL;
  }
  lin::Linear* L = new (std::nothrow) lin::Linear;
  if (!L) {
    set_error("asap_fp8_linear_register: out of host memory");
    return ASAP_EINVAL;
  }
  // the kernels are loaded here, not by a first call that may be a captured one
  if (int rc = lin::ensure_attrs()) {
    delete L;
    return rc;
  }
  for (int split = 1; split <= lin::SK_MAX_SPLIT; split *= 2) lin::clusters_at_once(split, false);
  L->d = *d;
  L->KB = (d->k + 127) / 128;
  L->NB = (d->n + 127) / 128;
  int rc = make_tmap_2d(&L->map, CU_TENSOR_MAP_DATA_TYPE_UINT8, (const void*)d->w, d->k, d->n, d->k, lin::BK, 128,
                        "linear weights");
  if (!rc) {
    try {
      std::lock_guard<std::mutex> lk(lin::g_mu);
      lin::g_linear[lin::g_next] = L;
      *handle = lin::g_next++;
      return ASAP_OK;
    } catch (...) {
      set_error("asap_fp8_linear_register: out of host memory");
      rc = ASAP_EINVAL;
    }
  }
  delete L;
  return rc;
}

int asap_fp8_linear_release(uint64_t handle) {
  std::lock_guard<std::mutex> lk(lin::g_mu);
  auto it = lin::g_linear.find(handle);
  if (it == lin::g_linear.end()) {
    set_error("asap_fp8_linear_release: unknown handle %llu", (unsigned long long)handle);
    return ASAP_EINVAL;
  }
  delete it->second;
  lin::g_linear.erase(it);
  return ASAP_OK;
}

uint64_t asap_fp8_linear_ws_bytes(int32_t m, int32_t k) {
  if (m < 1 || m > ASAP_LINEAR_MAX_ROWS || k < 1 || k > ASAP_LINEAR_MAX_DIM) return 0;
  if (m <= lin::kInKernelRows && k <= lin::kInKernelDim) return 0;
  const lin::ActWs a = lin::act_ws(m, k);
  return a.codes + a.scales;
}

int asap_fp8_linear(uint64_t handle, uint64_t x, int64_t ldx, int32_t m, int32_t fp16, uint64_t out, uint64_t ws,
                    uint64_t ws_bytes, uint64_t status, uint64_t timeout_ns, void* stream) {
  const lin::Linear* L = lin::find(handle);
  if (!L) {
    set_error("asap_fp8_linear: unknown handle %llu", (unsigned long long)handle);
    return ASAP_EINVAL;
  }
  const uint64_t need = asap_fp8_linear_ws_bytes(m, L->d.k);
  if (int rc = lin::check_rows("asap_fp8_linear", m, x, ldx, L->d.k, out, ws, ws_bytes, need)) return rc;
  if (int rc = lin::ensure_attrs()) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  const lin::ActWs a = lin::act_ws(m, L->d.k);
  lin::SkinnyParams p = lin::skinny_params(x, ldx, m, fp16, a.mp, status, timeout_ns);
  p.out = (void*)out;
  if (m <= lin::kInKernelRows && L->d.k <= lin::kInKernelDim) {
    const lin::SkinnyPlan pl = lin::skinny_plan<0, 0>(L, m);
    if (!pl) {
      set_error("asap_fp8_linear: no launch for %d rows of %d", m, L->d.k);
      return ASAP_EINVAL;
    }
    return lin::skinny<0, 0>(L, pl, p, 0, 0, st);
  }
  const lin::SkinnyPlan pl = lin::skinny_plan<0, 1>(L, m);
  if (pl && pl.rounds < lin::tile_rounds(L, false, m)) {
    if (int rc = lin::quantise(x, ldx, m, L, fp16, false, ws, ws + a.codes, a.mp, st)) return rc;
    return lin::skinny<0, 1>(L, pl, p, ws, ws + a.codes, st);
  }
  if (int rc = lin::quantise(x, ldx, m, L, fp16, L->d.atoms != 0, ws, ws + a.codes, a.mp, st)) return rc;
  return lin::product(L, false, ws, ws + a.codes, m, a.mp, out, L->d.n, fp16, 0.f, 0, 0, status, timeout_ns, st);
}

uint64_t asap_fp8_shared_ws_bytes(int32_t m, int32_t hidden, int32_t inter) {
  if (m < 1 || m > ASAP_LINEAR_MAX_ROWS || hidden < 1 || hidden > ASAP_LINEAR_MAX_DIM || inter < 1 ||
      inter > ASAP_LINEAR_MAX_DIM)
    return 0;
  const lin::ActWs a = lin::act_ws(m, hidden), b = lin::act_ws(m, inter);
  return a.codes + a.scales + b.codes + b.scales;
}

int asap_fp8_shared(uint64_t w13_handle, uint64_t w2_handle, uint64_t x, int64_t ldx, int32_t m, int32_t fp16,
                    float swiglu_limit, uint64_t out, uint64_t ws, uint64_t ws_bytes, uint64_t status,
                    uint64_t timeout_ns, void* stream) {
  const lin::Linear *L13 = lin::find(w13_handle), *L2 = lin::find(w2_handle);
  if (!L13 || !L2) {
    set_error("asap_fp8_shared: unknown handle %llu / %llu", (unsigned long long)w13_handle,
              (unsigned long long)w2_handle);
    return ASAP_EINVAL;
  }
  if (L13->d.n % 256 || L2->d.k != L13->d.n / 2 || L2->d.n != L13->d.k || !L13->d.atoms != !L2->d.atoms) {
    set_error("asap_fp8_shared: w13 [%d, %d] and w2 [%d, %d] are not [2I, H] and [H, I] with I %% 128 == 0 and scales "
              "of one kind", L13->d.n, L13->d.k, L2->d.n, L2->d.k);
    return ASAP_EINVAL;
  }
  const int32_t H = L13->d.k, I = L2->d.k;
  const uint64_t need = asap_fp8_shared_ws_bytes(m, H, I);
  if (int rc = lin::check_rows("asap_fp8_shared", m, x, ldx, H, out, ws, ws_bytes, need)) return rc;
  if (int rc = lin::ensure_attrs()) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  const lin::ActWs a = lin::act_ws(m, H), b = lin::act_ws(m, I);
  const uint64_t sa = ws + a.codes, hq = sa + a.scales, sh = hq + b.codes;
  const lin::SkinnyPlan up = lin::skinny_plan<1, 1>(L13, m), down = lin::skinny_plan<0, 1>(L2, m);
  if (up && down && up.rounds + down.rounds < lin::tile_rounds(L13, true, m) + lin::tile_rounds(L2, false, m)) {
    lin::SkinnyParams p = lin::skinny_params(x, ldx, m, fp16, a.mp, status, timeout_ns);
    p.swiglu_limit = swiglu_limit;
    p.out_q = (uint8_t*)hq;
    p.out_sa = (float*)sh;
    p.out = (void*)out;
    if (int rc = lin::quantise(x, ldx, m, L13, fp16, false, ws, sa, a.mp, st)) return rc;
    if (int rc = lin::skinny<1, 1>(L13, up, p, ws, sa, st)) return rc;
    return lin::skinny<0, 1>(L2, down, p, hq, sh, st);
  }
  if (int rc = lin::quantise(x, ldx, m, L13, fp16, L13->d.atoms != 0, ws, sa, a.mp, st)) return rc;
  if (int rc = lin::product(L13, true, ws, sa, m, a.mp, 0, 0, fp16, swiglu_limit, hq, sh, status, timeout_ns, st))
    return rc;
  return lin::product(L2, false, hq, sh, m, b.mp, out, H, fp16, 0.f, 0, 0, status, timeout_ns, st);
}

}  // extern "C"
