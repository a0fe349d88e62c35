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

__device__ __forceinline__ float swiglu(float g, float u, float limit) {
  if (limit > 0.f) {
    g = fminf(g, limit);
    u = fminf(fmaxf(u, -limit), limit);
  }
  return g / (1.f + expf(-g)) * u;
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
  int32_t M, K, KB, fp16, pow2;
  int64_t mp;
  uint8_t* xq;
  float* sa;
};

constexpr int QUANT_AHEAD = 4;
__global__ void __launch_bounds__(256) quant_rows_kernel(const __grid_constant__ QuantArgs p) {
  const int lane = threadIdx.x & 31;
  const int chunks = (p.KB + 1) / 2;  // of 256 values
  const int64_t items = (int64_t)p.M * chunks, step = (int64_t)gridDim.x * (blockDim.x >> 5);
  for (int64_t i0 = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); i0 < items; i0 += QUANT_AHEAD * step) {
    uint4 u[QUANT_AHEAD];
    int64_t row[QUANT_AHEAD];
    int col[QUANT_AHEAD];
#pragma unroll
    for (int j = 0; j < QUANT_AHEAD; ++j) {
      const int64_t i = i0 + j * step;
      row[j] = i / chunks;
      col[j] = (int)(i - row[j] * chunks) * 256 + lane * 8;
      u[j] = make_uint4(0, 0, 0, 0);
      if (i < items && col[j] < p.K) u[j] = *reinterpret_cast<const uint4*>(p.x + row[j] * p.ldx + col[j]);
    }
#pragma unroll
    for (int j = 0; j < QUANT_AHEAD; ++j) {
      uint2 codes;
      float scale;
      quant8(u[j], p.fp16 != 0, p.pow2 != 0, codes, scale);
      if (i0 + j * step < items && col[j] < p.KB * 128) {
        *reinterpret_cast<uint2*>(p.xq + row[j] * p.KB * 128 + col[j]) = codes;
        if ((lane & 15) == 0) {
          const int kb = col[j] / 128;
          if (p.pow2)
            *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(p.sa) + atom_off(row[j], kb, p.KB)) =
                atom_word(scale);
          else p.sa[(int64_t)kb * p.mp + row[j]] = scale;
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
  ASAP_CUDA(cudaFuncSetAttribute(linear_gemm_kernel<1>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
  ASAP_CUDA(cudaFuncSetAttribute(linear_pow2_kernel<0>, cudaFuncAttributeMaxDynamicSharedMemorySize, P2_SMEM_BYTES));
  ASAP_CUDA(cudaFuncSetAttribute(linear_pow2_kernel<1>, cudaFuncAttributeMaxDynamicSharedMemorySize, P2_SMEM_BYTES));
  for (const void* f : {(const void*)linear_skinny_kernel<16, 0>, (const void*)linear_skinny_kernel<32, 0>,
                        (const void*)linear_skinny_kernel<64, 0>, (const void*)linear_skinny_kernel<128, 0>,
                        (const void*)linear_skinny_kernel<16, 1>, (const void*)linear_skinny_kernel<32, 1>,
                        (const void*)linear_skinny_kernel<64, 1>})
    ASAP_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem));
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
  if (!out || (out & 15) || !ws || (ws & 255) || have < need) {
    set_error("%s: out must be 16-byte and the workspace 256-byte aligned and hold %llu bytes (got %llu)", fn,
              (unsigned long long)need, (unsigned long long)have);
    return ASAP_EINVAL;
  }
  return ASAP_OK;
}

static int quantise(uint64_t x, int64_t ldx, int32_t m, const Linear* L, int32_t fp16, uint64_t xq, uint64_t sa,
                    int64_t mp, cudaStream_t st) {
  QuantArgs q{};
  q.x = (const uint16_t*)x;
  q.ldx = ldx;
  q.M = m;
  q.K = L->d.k;
  q.KB = L->KB;
  q.fp16 = fp16;
  q.pow2 = L->d.atoms != 0;
  q.mp = mp;
  q.xq = (uint8_t*)xq;
  q.sa = (float*)sa;
  const int64_t items = (int64_t)m * ((L->KB + 1) / 2);
  const int64_t blocks = (items + 7) / 8, cap = 8ll * sm_count();
  quant_rows_kernel<<<(int)(blocks < cap ? blocks : cap), 256, 0, st>>>(q);
  ASAP_CHECK_LAUNCH("quant_rows_kernel");
  return ASAP_OK;
}

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
  const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles;
  const int grid = (int)(tiles < sm_count() ? tiles : sm_count());
  if (L->d.atoms) {
    if (swiglu) linear_pow2_kernel<1><<<grid, P2_THREADS, P2_SMEM_BYTES, st>>>(p);
    else linear_pow2_kernel<0><<<grid, P2_THREADS, P2_SMEM_BYTES, st>>>(p);
    ASAP_CHECK_LAUNCH("linear_pow2_kernel");
    return ASAP_OK;
  }
  if (swiglu) linear_gemm_kernel<1><<<grid, THREADS, SMEM_BYTES, st>>>(p);
  else linear_gemm_kernel<0><<<grid, THREADS, SMEM_BYTES, st>>>(p);
  ASAP_CHECK_LAUNCH("linear_gemm_kernel");
  return ASAP_OK;
}

// ------------------------------------------------------------------ few rows
// How a product of few rows is launched, or split = 0: not at all.
struct SkinnyPlan {
  int tn, split, stages, max_kb, smem;
};

// TN is the smallest of 16, 32, 64, 128 that holds the rows (64 at most with SwiGLU, whose tiles are two), halved while
// a CTA's part of x does not fit beside the fewest stages.  K is split as far as the grid stays within two CTAs per SM.
template <int SWIGLU>
static SkinnyPlan skinny_plan(const Linear* L, int32_t m) {
  const int n_tiles = SWIGLU ? L->d.n / 256 : (L->d.n + 127) / 128;
  int tn = m <= 16 ? 16 : m <= 32 ? 32 : (m <= 64 || SWIGLU) ? 64 : 128;
  for (; tn >= 16; tn /= 2) {
    const int64_t y = (m + tn - 1) / tn;
    int split = 1;
    while (split < SK_MAX_SPLIT && 2 * split <= L->KB && n_tiles * y * split * 2 <= 2 * sm_count()) split *= 2;
    for (; split <= SK_MAX_SPLIT && split <= L->KB; split *= 2) {
      SkinnyPlan pl;
      pl.tn = tn;
      pl.split = split;
      pl.max_kb = (L->KB + split - 1) / split;
      const int tiles = SWIGLU ? 2 : 1, stage = tiles * 128 * BK, part = tiles * tn * 512;
      const int least = part > 3 * stage ? (part + stage - 1) / stage : 3;
      const int fixed = 1024 + 2048 + pl.max_kb * (tn * BK + tn * 4 + 8);
      if (pl.max_kb > SK_MAX_KB || fixed + least * stage > kMaxSmem) continue;
      // half an SM's shared memory if three stages fit it, so that two CTAs share the SM
      const int half = kMaxSmem / 2 - 1024;
      const int room = tiles * tn <= 64 && fixed + least * stage <= half ? half : kMaxSmem;
      pl.stages = (room - fixed) / stage;
      if (pl.stages > SK_MAX_STAGES) pl.stages = SK_MAX_STAGES;
      if (pl.stages > pl.max_kb) pl.stages = pl.max_kb;
      if (pl.stages < least) pl.stages = least;
      pl.smem = fixed + pl.stages * stage;
      // never three CTAs on an SM: the third would wait for tensor memory while its cluster waits for it
      if (pl.smem < 80 * 1024) pl.smem = 80 * 1024;
      return pl;
    }
  }
  return SkinnyPlan{0, 0, 0, 0, 0};
}

template <int SWIGLU>
static int skinny(const Linear* L, const SkinnyPlan& pl, SkinnyParams& p, cudaStream_t st) {
  p.tmap_w = L->map;
  p.K = L->d.k;
  p.N = L->d.n;
  p.KB = L->KB;
  p.NB = L->NB;
  p.split = pl.split;
  p.stages = pl.stages;
  p.max_kb = pl.max_kb;
  p.sb = (const float*)L->d.scale;
  p.pow2 = L->d.atoms != 0;
  const int n_tiles = SWIGLU ? L->d.n / 256 : (L->d.n + 127) / 128;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(n_tiles * pl.split, (p.M + pl.tn - 1) / pl.tn);
  cfg.blockDim = dim3(SK_THREADS);
  cfg.dynamicSmemBytes = pl.smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = pl.split;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (pl.tn == 16) ASAP_CUDA(cudaLaunchKernelEx(&cfg, linear_skinny_kernel<16, SWIGLU>, p));
  else if (pl.tn == 32) ASAP_CUDA(cudaLaunchKernelEx(&cfg, linear_skinny_kernel<32, SWIGLU>, p));
  else if (pl.tn == 64) ASAP_CUDA(cudaLaunchKernelEx(&cfg, linear_skinny_kernel<64, SWIGLU>, p));
  else if constexpr (!SWIGLU) ASAP_CUDA(cudaLaunchKernelEx(&cfg, linear_skinny_kernel<128, 0>, p));
  return ASAP_OK;
}

constexpr int kSkinnyRows = 64;  // at most this many rows take the few-rows kernel

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
  if (m <= lin::kSkinnyRows) {
    const lin::SkinnyPlan pl = lin::skinny_plan<0>(L, m);
    if (pl.split) {
      lin::SkinnyParams p{};
      p.x = (const uint16_t*)x;
      p.ldx = ldx;
      p.M = m;
      p.fp16 = fp16;
      p.out = (void*)out;
      p.status = status;
      p.timeout_ns = timeout_ns;
      return lin::skinny<0>(L, pl, p, st);
    }
  }
  const lin::ActWs a = lin::act_ws(m, L->d.k);
  if (int rc = lin::quantise(x, ldx, m, L, fp16, ws, ws + a.codes, a.mp, st)) return rc;
  return lin::product(L, false, ws, ws + a.codes, m, a.mp, out, L->d.n, fp16, 0.f, 0, 0, status, timeout_ns, st);
}

uint64_t asap_fp8_shared_ws_bytes(int32_t m, int32_t hidden, int32_t inter) {
  const uint64_t a = asap_fp8_linear_ws_bytes(m, hidden), b = asap_fp8_linear_ws_bytes(m, inter);
  return a && b ? a + b : 0;
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
  if (m <= lin::kSkinnyRows) {
    const lin::SkinnyPlan up = lin::skinny_plan<1>(L13, m), down = lin::skinny_plan<0>(L2, m);
    if (up.split && down.split) {
      lin::SkinnyParams p{};
      p.x = (const uint16_t*)x;
      p.ldx = ldx;
      p.M = m;
      p.fp16 = fp16;
      p.swiglu_limit = swiglu_limit;
      p.out_q = (uint8_t*)hq;
      p.out_sa = (float*)sh;
      p.mp = b.mp;
      p.status = status;
      p.timeout_ns = timeout_ns;
      if (int rc = lin::skinny<1>(L13, up, p, st)) return rc;
      p.x = nullptr;
      p.xq = (const uint8_t*)hq;
      p.sa = (const float*)sh;
      p.out = (void*)out;
      return lin::skinny<0>(L2, down, p, st);
    }
  }
  if (int rc = lin::quantise(x, ldx, m, L13, fp16, ws, sa, a.mp, st)) return rc;
  if (int rc = lin::product(L13, true, ws, sa, m, a.mp, 0, 0, fp16, swiglu_limit, hq, sh, status, timeout_ns, st))
    return rc;
  return lin::product(L2, false, hq, sh, m, b.mp, out, H, fp16, 0.f, 0, 0, status, timeout_ns, st);
}

}  // extern "C"
