// The vocabulary head in 8-bit integers: hidden states quantised per token, times a weight whose
// rows (vocabulary entries) are 8-bit codes with one scale each.
//
//   frx_quantize_i8      scale_r = fl32(max_k |x_rk| / 127),  code_rk = nearest integer to
//                        x_rk / scale_r (ties to even)
//   frx_gemm_i8          y[r, j] = (sum_k code_rk w_jk) scale_r wscale_j + bias_j
//   frx_i8_ce_entropy    the same product reduced to softmax partials (m, s, u, zt) by the epilogue, and
//                        those to cross-entropy, entropy and log-probability per row
//
// |code| <= 127, so a sum over K <= 131072 products stays below 2^31: the int32 accumulators of
// kind::i8 hold it exactly and the result does not depend on the order of the products.
#include <cstring>
#include <type_traits>

#include "frx_epilogue.cuh"
#include "frx_host.cuh"

namespace frx {

constexpr int64_t kI8MaxK = 131072;

// ------------------------------------------------------------------------------------ quantisation
// Eight consecutive values of a row as they lie in memory, and as floats.
template <typename T>
struct Raw8 {  // 16-bit types
  uint4 q;
  __device__ void load(const T* p) { q = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ void floats(float (&v)[8]) const {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2(w[i], std::is_same<T, __half>::value);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
};
template <>
struct Raw8<float> {
  float4 a, b;
  __device__ void load(const float* p) {
    a = __ldg(reinterpret_cast<const float4*>(p));
    b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  }
  __device__ void floats(float (&v)[8]) const {
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
};

__device__ __forceinline__ float one_f32(const float* p) { return __ldg(p); }
__device__ __forceinline__ float one_f32(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float one_f32(const __half* p) { return __half2float(*p); }

// Running |x| maximum that keeps NaN (fmaxf drops it): a row with NaN or infinity must show.
__device__ __forceinline__ float amax_nan(float a, float x) {
  x = fabsf(x);
  return (x > a || x != x) ? x : a;
}

// The row's scale and 1 / scale: scale = max / 127 rounded once; 0 for a row whose scale is below 2^-120
// (its codes are 0; q8_code's FMA would lose bits to underflow there), NaN for a row with NaN or
// infinity (its codes are 0 too).
__device__ __forceinline__ void q8_scale(float amax, float& scale, float& inv) {
  scale = __fdiv_rn(amax, 127.0f);
  inv = 0.0f;
  if (!(amax <= 3.402823466e38f))
    scale = __int_as_float(0x7fc00000);
  else if (scale < 7.52316385e-37f)
    scale = 0.0f;
  else
    inv = __frcp_rn(scale);
}

// Nearest integer to the real quotient x / scale, ties to even. x * inv is within 127 * 2^-22 of it, so
// its rounding is right unless it lands within 1e-4 of a half; there the sign of x - half * scale, exact
// from one FMA, decides.
__device__ __forceinline__ int q8_code(float x, float scale, float inv) {
  const float y = x * inv;
  float k = rintf(y);
  if (fabsf(y - k) > 0.4999f) {
    const float lo = floorf(y);
    const float r = fmaf(-(lo + 0.5f), scale, x);  // sign of x / scale - (lo + 1/2)
    const float even = 2.0f * rintf(0.5f * (lo + 0.5f));
    k = r > 0.0f ? lo + 1.0f : (r < 0.0f ? lo : even);
  }
  return static_cast<int>(k);
}

__device__ __forceinline__ uint32_t pack4_i8(int a, int b, int c, int d) {
  return (a & 0xFF) | ((b & 0xFF) << 8) | ((c & 0xFF) << 16) | (static_cast<uint32_t>(d) << 24);
}

constexpr int kQ8Threads = 256;

// A row belongs to kLanes threads (a warp, or the whole CTA). The row's first 8 * kLanes * kHeld values stay
// in registers between the maximum and the codes, so such a row is read once, with all its loads in flight
// together; what is longer is read again.
template <typename T, int kLanes, int kHeld>
__global__ void __launch_bounds__(kQ8Threads)
    quantize_i8_kernel(const T* __restrict__ x, int64_t ld_x, int64_t rows, int64_t cols, int8_t* __restrict__ codes,
                       int64_t ld_codes, float* __restrict__ scale_out, int vec_ok) {
  grid_dep_launch();
  __shared__ float red[kQ8Threads / 32];
  constexpr int kRows = kQ8Threads / kLanes;
  const int t = threadIdx.x % kLanes;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kLanes;
  if (kLanes == 32 && row >= rows) return;
  const T* xr = x + row * ld_x;
  int8_t* cr = codes + row * ld_codes;
  const int64_t nv = vec_ok ? cols / 8 : 0;
  Raw8<T> held[kHeld];
  float v[8];
  float amax = 0.0f;
#pragma unroll
  for (int h = 0; h < kHeld; ++h)
    if (t + h * kLanes < nv) held[h].load(xr + 8 * (t + h * kLanes));
#pragma unroll
  for (int h = 0; h < kHeld; ++h) {
    if (t + h * kLanes < nv) {
      held[h].floats(v);
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = amax_nan(amax, v[j]);
    }
  }
  for (int64_t i = t + kHeld * kLanes; i < nv; i += kLanes) {
    Raw8<T> r;
    r.load(xr + 8 * i);
    r.floats(v);
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = amax_nan(amax, v[j]);
  }
  for (int64_t i = 8 * nv + t; i < cols; i += kLanes) amax = amax_nan(amax, one_f32(xr + i));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = amax_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if (kLanes > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kQ8Threads / 32; ++w) amax = amax_nan(amax, red[w]);
  }
  float scale, inv;
  q8_scale(amax, scale, inv);
  if (t == 0) scale_out[row] = scale;
  const bool live = inv != 0.0f;
  auto put8 = [&](int64_t i) {
    int k[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) k[j] = live ? q8_code(v[j], scale, inv) : 0;
    *reinterpret_cast<uint2*>(cr + 8 * i) =
        make_uint2(pack4_i8(k[0], k[1], k[2], k[3]), pack4_i8(k[4], k[5], k[6], k[7]));
  };
#pragma unroll
  for (int h = 0; h < kHeld; ++h) {
    if (t + h * kLanes < nv) {
      held[h].floats(v);
      put8(t + h * kLanes);
    }
  }
  for (int64_t i = t + kHeld * kLanes; i < nv; i += kLanes) {
    Raw8<T> r;
    r.load(xr + 8 * i);
    r.floats(v);
    put8(i);
  }
  for (int64_t i = 8 * nv + t; i < cols; i += kLanes)
    cr[i] = static_cast<int8_t>(live ? q8_code(one_f32(xr + i), scale, inv) : 0);
}

// ------------------------------------------------------------------------------------ epilogues
// One value of an optional bias vector (bf16, fp16 or fp32).
__device__ __forceinline__ float bias_at(const void* bias, int dtype, int64_t i) {
  if (dtype == FRX_DTYPE_F32) return __ldg(static_cast<const float*>(bias) + i);
  return unpack2(__ldg(static_cast<const uint16_t*>(bias) + i), dtype == FRX_DTYPE_F16).x;
}

template <typename OutT>
__device__ __forceinline__ OutT round_out(float y);
template <>
__device__ __forceinline__ float round_out<float>(float y) { return y; }
template <>
__device__ __forceinline__ __nv_bfloat16 round_out<__nv_bfloat16>(float y) { return __float2bfloat16_rn(y); }
template <>
__device__ __forceinline__ __half round_out<__half>(float y) { return __float2half_rn(y); }

struct I8Out {
  const float* row_scale;  // [rows] of the tokens
  const float* col_scale;  // [cols] of the weight's rows
  const void* bias;
  int bias_dtype;
  void* out;
  int64_t ld_out;
  int rows;
  int cols;
};

// Stores vocabulary entry j (this lane's) of the 32 tokens from r: 32 neighbouring outputs per warp and token,
// coalesced rows without staging, whatever the output's alignment. s_scale: this warp's 32 floats of
// shared memory, through which every lane gets the tokens' scales.
template <typename OutT>
__device__ __forceinline__ void store_tokens32(const I8Out& p, const float (&v)[32], float* s_scale, int j, int r,
                                               float ws, float b, int lane) {
  const int lim = p.rows - r;
  __syncwarp();
  s_scale[lane] = lane < lim ? ld_dep_f32(p.row_scale + r + lane) : 0.0f;
  __syncwarp();
  OutT* dst = static_cast<OutT*>(p.out) + static_cast<int64_t>(r) * p.ld_out + j;
  const bool ok = j < p.cols;
  if (lim >= 32) {
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      const float4 xs = *reinterpret_cast<const float4*>(s_scale + i);
      const float f[4] = {xs.x, xs.y, xs.z, xs.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const OutT y = round_out<OutT>(fmaf(static_cast<float>(__float_as_int(v[i + k])) * f[k], ws, b));
        if (ok) dst[(i + k) * p.ld_out] = y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const OutT y = round_out<OutT>(fmaf(static_cast<float>(__float_as_int(v[i])) * s_scale[i], ws, b));
      if (ok && i < lim) dst[i * p.ld_out] = y;
    }
  }
}

// Output tile of the plain product on the CTA-pair core. The weight is the A operand, so a thread owns one
// vocabulary entry (TMEM lane).
template <typename OutT>
struct Int8StoreEpilogue {
  static constexpr int kSmemPerWarp = 128;
  static constexpr int kSmemBytes = 8 * kSmemPerWarp;
  using Params = I8Out;

  template <class Release>
  __device__ __forceinline__ static void run(const Params& p, uint8_t* stage, uint32_t tacc, int m_blk, int n_blk,
                                             int q, int lane, Release release) {
    const int j = m_blk * kBM + q * 32 + lane;  // vocabulary entry
    const int r0 = n_blk * kBN;                 // first token
    const int ntok = min(kBN, p.rows - r0);
    if (j - lane < p.cols) {
      const bool ok = j < p.cols;
      const float ws = ok ? __ldg(p.col_scale + j) : 0.0f;
      const float b = ok && p.bias != nullptr ? bias_at(p.bias, p.bias_dtype, j) : 0.0f;
      float v[32];
#pragma unroll 1
      for (int c = 0; c < ntok; c += 32) {
        __syncwarp();
        tmem_load_32cols(tacc + static_cast<uint32_t>(c), v);
        store_tokens32<OutT>(p, v, reinterpret_cast<float*>(stage), j, r0 + c, ws, b, lane);
      }
    }
    release();
  }

  __device__ __forceinline__ static void finish(const Params&, int) {}
};

// Softmax partials of the scaled product, in one pass over the accumulator: thread = token (TMEM lane), 32
// columns at a time with a running maximum, and s and u rescaled when it rises. Without a bias the token's
// scale xs > 0 is taken out: with y = acc * wscale, z = xs y has its maximum where y has, exp(z - m) =
// 2^((y - max y) xs log2 e), u = xs sum (y - max y) e. Pairs of columns share fp32x2 instructions; a column
// costs about 6 issue slots, of which the conversion of its int32 and its exponential go to the
// low-throughput unit.
template <bool kBias>
struct Int8CEPartialsEpilogue {
  // 32 weight scales and 32 bias values of the current columns
  static constexpr int kSmemPerWarp = 256;
  static constexpr int kSmemBytes = 8 * kSmemPerWarp;

  struct Params {
    const float* row_scale;
    const float* col_scale;
    const void* bias;
    int bias_dtype;
    const int64_t* target;
    int rows;
    int vocab_shard;
    float4* partials;
    int64_t tile_stride;
    int n_tiles;
    int* status;
  };

  template <class Release>
  __device__ __forceinline__ static void run(const Params& p, uint8_t* stage, uint32_t tacc, int m_blk, int n_blk,
                                             int q, int lane, Release release) {
    constexpr float kLow = -1e38f;  // below every logit; differences to it stay finite
    const int row0 = m_blk * kBM + q * 32;
    const int row = row0 + lane;
    if (row0 >= p.rows) {
      release();
      return;
    }
    const int n0 = n_blk * kBN;
    const int ncols = min(kBN, p.vocab_shard - n0);
    const bool row_ok = row < p.rows;
    const float xs = row_ok ? ld_dep_f32(p.row_scale + row) : 0.0f;
    // a negative scale (from the caller) turns the order round: then y = -acc * wscale with |xs|
    const bool flip = !kBias && __any_sync(0xffffffffu, xs < 0.0f);
    const float sign = xs < 0.0f ? -1.0f : 1.0f;
    const float f = kBias ? 1.0f : fabsf(xs);
    const float k = f * kLog2e;
    const uint64_t k2 = pack_f32x2(k, k), xs2 = pack_f32x2(xs, xs);
    int tcol = -1;
    if (row_ok && p.target != nullptr) {
      const long long lt = static_cast<long long>(p.target[row]) - n0;
      if (lt >= 0 && lt < ncols) tcol = static_cast<int>(lt);
    }
    float* s_ws = reinterpret_cast<float*>(stage);
    float* s_b = s_ws + 32;
    float ws = 0.0f, b = 0.0f;
    auto fetch = [&](int c) {
      const int col = c * 32 + lane;
      ws = col < ncols ? __ldg(p.col_scale + n0 + col) : 0.0f;
      if (kBias) b = col < ncols ? bias_at(p.bias, p.bias_dtype, n0 + col) : 0.0f;
    };
    fetch(0);
    float v[32];
    float m = kLow, zt = 0.0f, s = 0.0f, u = 0.0f;
#pragma unroll 1
    for (int c = 0; c * 32 < ncols; ++c) {
      const int lim = ncols - c * 32;
      __syncwarp();
      s_ws[lane] = ws;
      if (kBias) s_b[lane] = b;
      __syncwarp();
      if (lim > 32) fetch(c + 1);
      tmem_load_32cols(tacc + static_cast<uint32_t>(c * 32), v);
      uint64_t y[16];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(s_ws + 4 * i);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int j = 4 * i + 2 * h;
          y[2 * i + h] = mul_f32x2(pack_f32x2(static_cast<float>(__float_as_int(v[j])),
                                              static_cast<float>(__float_as_int(v[j + 1]))), h == 0 ? w.x : w.y);
        }
        if (kBias) {
          const ulonglong2 bb = *reinterpret_cast<const ulonglong2*>(s_b + 4 * i);
          y[2 * i] = fma_f32x2(y[2 * i], xs2, bb.x);
          y[2 * i + 1] = fma_f32x2(y[2 * i + 1], xs2, bb.y);
        }
      }
      if (flip) {
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = mul_f32x2(y[i], pack_f32x2(sign, sign));
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) unpack_f32x2(y[i], v[2 * i], v[2 * i + 1]);
      if (lim < 32) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j >= lim) v[j] = kLow;
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = pack_f32x2(v[2 * i], v[2 * i + 1]);
      }
      if ((tcol >> 5) == c) zt = select32(v, tcol & 31);
      float top = m;
#pragma unroll
      for (int j = 0; j < 32; j += 2) top = fmaxf(top, fmaxf(v[j], v[j + 1]));
      const float d = m - top;
      const float r = ex2_approx(d * k);
      u = fmaf(d, s, u) * r;
      s *= r;
      m = top;
      const uint64_t neg = pack_f32x2(-top, -top);
      uint64_t s2[2] = {0, 0}, u2[2] = {0, 0};
      auto add = [&](int i, float live0, float live1) {
        const uint64_t dd = add_f32x2(y[i], neg);
        float a0, a1;
        unpack_f32x2(mul_f32x2(dd, k2), a0, a1);
        const uint64_t e = pack_f32x2(ex2_approx(a0) * live0, ex2_approx(a1) * live1);
        s2[i & 1] = add_f32x2(s2[i & 1], e);
        u2[i & 1] = fma_f32x2(dd, e, u2[i & 1]);
      };
      if (lim >= 32) {
#pragma unroll
        for (int i = 0; i < 16; ++i) add(i, 1.0f, 1.0f);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) add(i, 2 * i < lim ? 1.0f : 0.0f, 2 * i + 1 < lim ? 1.0f : 0.0f);
      }
      float f0, f1;
      unpack_f32x2(add_f32x2(s2[0], s2[1]), f0, f1);
      s += f0 + f1;
      unpack_f32x2(add_f32x2(u2[0], u2[1]), f0, f1);
      u += f0 + f1;
    }
    release();
    if (row_ok && device_check(n_blk < p.n_tiles, p.status)) {
      p.partials[static_cast<int64_t>(n_blk) * p.tile_stride + row] = make_float4(m * f, s, u * f, zt * f);
    }
  }

  __device__ __forceinline__ static void finish(const Params&, int) {}
};

// ------------------------------------------------------------------------------------ few tokens
// Up to 128 tokens: the product streams the weight once and is bound by HBM. A CTA owns 128 vocabulary entries
// (the M of the MMA) against all tokens (its N, rounded up to 16), so the padding of the tokens costs nothing in
// HBM, and two CTAs per SM keep up to 2 x 96 KiB of weight in flight through rings of 128-byte deep K steps.
// The first ring of weight tiles is requested before the wait for the tokens' quantisation.
constexpr int kFewThreads = 192;
constexpr int kFewMaxTokens = 128;
constexpr int kFewWBytes = 128 * 128;
constexpr int kFewMaxStages = 6;
constexpr int kFewRingBytes = 108 * 1024;

inline int few_tokens_padded(int64_t rows) { return static_cast<int>((rows + 15) / 16 * 16); }
inline int few_stages(int nt) {
  const int n = kFewRingBytes / (kFewWBytes + nt * 128);
  return n < kFewMaxStages ? n : kFewMaxStages;
}

template <typename OutT>
__global__ void __launch_bounds__(kFewThreads, 2)
    gemm_i8_few_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                       const __grid_constant__ I8Out p, int nt, int num_k, int stages, int* status) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int x_bytes = nt * 128;
  uint8_t* s_w = smem;
  uint8_t* s_x = smem + stages * kFewWBytes;
  float* s_scale = reinterpret_cast<float*>(s_x + stages * x_bytes);  // 32 per epilogue warp
  uint64_t* full = reinterpret_cast<uint64_t*>(s_scale + 128);
  uint64_t* empty = full + kFewMaxStages;
  uint64_t* done = empty + kFewMaxStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  if (!device_check(reinterpret_cast<const uint8_t*>(tmem_slot + 2) - smem_raw <=
                        static_cast<ptrdiff_t>(dynamic_smem_bytes()),
                    threadIdx.x == 0 ? status : nullptr))
    return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = static_cast<int>(blockIdx.x) * 128;
  const uint32_t tmem_cols = nt <= 32 ? 32u : (nt <= 64 ? 64u : 128u);
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_x);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      const int pre = num_k < stages ? num_k : stages;
      for (int kb = 0; kb < pre; ++kb) {
        mbar_arrive_expect_tx(&full[kb], static_cast<uint32_t>(kFewWBytes + x_bytes));
        tma_load_2d(s_w + kb * kFewWBytes, &tm_w, &full[kb], kb * 128, n0);
      }
      grid_dep_wait();
      for (int kb = 0; kb < pre; ++kb) tma_load_2d(s_x + kb * x_bytes, &tm_x, &full[kb], kb * 128, 0);
      int stage = 0;
      uint32_t phase = 0;  // of empty[stage] to wait for
      int kb = pre;
      for (; kb < num_k; ++kb) {
        if (!mbar_wait_bounded(&empty[stage], phase, abort_flag, status, kStatusTimeoutProducer)) break;
        mbar_arrive_expect_tx(&full[stage], static_cast<uint32_t>(kFewWBytes + x_bytes));
        tma_load_2d(s_w + stage * kFewWBytes, &tm_w, &full[stage], kb * 128, n0);
        tma_load_2d(s_x + stage * x_bytes, &tm_x, &full[stage], kb * 128, 0);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (kb < num_k) {
        // gave up: let every copy still in flight land before the shared memory goes away
        for (int j = kb > stages ? kb - stages : 0; j < kb; ++j)
          mbar_wait_drain(&full[j % stages], static_cast<uint32_t>((j / stages) & 1), status);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = make_idesc_i8(128, nt);
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = 0; kb < num_k; ++kb) {
        if (!mbar_wait_bounded(&full[stage], phase, abort_flag, status, kStatusTimeoutMma)) break;
        tc_fence_after();
        const uint32_t w_addr = smem_u32(s_w + stage * kFewWBytes);
        const uint32_t x_addr = smem_u32(s_x + stage * x_bytes);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_i8(tmem, make_smem_desc_sw128(w_addr + k * 32, 16, 1024), make_smem_desc_sw128(x_addr + k * 32, 16, 1024),
                  idesc, (kb | k) != 0 ? 1u : 0u);
        umma_commit(&empty[stage]);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      umma_commit(done);
      mbar_wait_drain(done, 0, status);  // before TMEM is released
    }
    __syncwarp();
  } else {
    const int q = warp & 3;
    const int j = n0 + q * 32 + lane;
    const bool ok = j < p.cols;
    const float ws = ok ? __ldg(p.col_scale + j) : 0.0f;
    const float b = ok && p.bias != nullptr ? bias_at(p.bias, p.bias_dtype, j) : 0.0f;
    grid_dep_wait();
    int good = 1;
    if (lane == 0)
      good = mbar_wait_bounded(done, 0, abort_flag, status, kStatusTimeoutEpilogue) && *abort_flag == 0 ? 1 : 0;
    good = __shfl_sync(0xffffffffu, good, 0);
    if (good && j - lane < p.cols) {
      tc_fence_after();
      const uint32_t tacc = tmem + (static_cast<uint32_t>(q * 32) << 16);
      float v[32];
#pragma unroll 1
      for (int c = 0; c < p.rows; c += 32) {
        __syncwarp();
        tmem_load_32cols(tacc + static_cast<uint32_t>(c), v);
        store_tokens32<OutT>(p, v, s_scale + q * 32, j, c, ws, b, lane);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
}

// ------------------------------------------------------------------------------------ host side
static bool is_float_dtype(int d) { return d == FRX_DTYPE_BF16 || d == FRX_DTYPE_F32 || d == FRX_DTYPE_F16; }

struct I8Operands {
  const int8_t* x;
  int64_t ld_x;
  const float* x_scale;
  const void* w;
  int64_t ld_w;
  const float* w_scale;
  const void* bias;
  int bias_dtype;
  int64_t rows, cols, k;
  bool quantised_here;  // the launch before the product wrote x and x_scale
};

inline int64_t round_up_to(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

// Rows from which each row is left to one warp instead of one CTA. Measured on rows of 4096 bf16 values: see
// frx_quantize_i8.
constexpr int64_t kQ8WarpRows = 1024;

template <typename T, int kHeldWarp>
static int launch_quantize(const void* x, int64_t ld_x, int64_t rows, int64_t cols, int8_t* codes, int64_t ld_codes,
                           float* scale, cudaStream_t stream) {
  const int vec_ok = aligned16(x) && (ld_x * sizeof(T)) % 16 == 0 && (reinterpret_cast<uintptr_t>(codes) & 7u) == 0 &&
                     ld_codes % 8 == 0;
  const T* xt = static_cast<const T*>(x);
  if (rows >= kQ8WarpRows) {
    constexpr int kRows = kQ8Threads / 32;
    quantize_i8_kernel<T, 32, kHeldWarp><<<static_cast<unsigned>((rows + kRows - 1) / kRows), kQ8Threads, 0, stream>>>(
        xt, ld_x, rows, cols, codes, ld_codes, scale, vec_ok);
  } else {
    quantize_i8_kernel<T, kQ8Threads, 4><<<static_cast<unsigned>(rows), kQ8Threads, 0, stream>>>(
        xt, ld_x, rows, cols, codes, ld_codes, scale, vec_ok);
  }
  FRX_CUDA_CHECK(cudaGetLastError());
  return FRX_OK;
}

static int quantize(const void* x, int dtype, int64_t ld_x, int64_t rows, int64_t cols, int8_t* codes,
                    int64_t ld_codes, float* scale, cudaStream_t stream) {
  if (dtype == FRX_DTYPE_F32) return launch_quantize<float, 8>(x, ld_x, rows, cols, codes, ld_codes, scale, stream);
  if (dtype == FRX_DTYPE_BF16)
    return launch_quantize<__nv_bfloat16, 16>(x, ld_x, rows, cols, codes, ld_codes, scale, stream);
  return launch_quantize<__half, 16>(x, ld_x, rows, cols, codes, ld_codes, scale, stream);
}

// Checks shared by the two products; floating-point tokens are quantised into the workspace, whose used
// part is returned in *used.
static int prepare_i8(const char* what, const void* x, int x_dtype, int64_t ld_x, const float* x_scale, const void* w,
                      int64_t ld_w, const float* w_scale, const void* bias, int bias_dtype, int64_t rows, int64_t cols,
                      int64_t k, void* workspace, int64_t workspace_bytes, I8Operands* op, int64_t* used,
                      int64_t more_bytes, cudaStream_t stream) {
  FRX_REQUIRE(rows >= 0 && cols >= 1 && k >= 1 && rows < (1ll << 31) && cols < (1ll << 31), FRX_ERR_INVALID_ARG,
              "%s: bad sizes rows=%lld cols=%lld k=%lld", what, (long long)rows, (long long)cols, (long long)k);
  FRX_REQUIRE(k <= kI8MaxK, FRX_ERR_UNSUPPORTED, "%s: k %lld > %lld could overflow the int32 accumulators", what,
              (long long)k, (long long)kI8MaxK);
  FRX_REQUIRE(x_dtype == FRX_DTYPE_I8 || is_float_dtype(x_dtype), FRX_ERR_INVALID_ARG, "%s: unknown x_dtype %d", what,
              x_dtype);
  if (rows == 0) return FRX_OK;
  const bool codes = x_dtype == FRX_DTYPE_I8;
  FRX_REQUIRE(x != nullptr && w != nullptr && w_scale != nullptr && (!codes || x_scale != nullptr),
              FRX_ERR_INVALID_ARG, "%s: null operand or scale pointer", what);
  FRX_REQUIRE(ld_x >= k && ld_w >= k && aligned16(w) && ld_w % 16 == 0 && (!codes || (aligned16(x) && ld_x % 16 == 0)),
              FRX_ERR_INVALID_ARG,
              "%s: codes need 16-byte aligned bases and leading dimensions >= k that are multiples of 16 (got %lld, "
              "%lld)", what, (long long)ld_x, (long long)ld_w);
  FRX_REQUIRE(bias == nullptr || is_float_dtype(bias_dtype), FRX_ERR_INVALID_ARG, "%s: unknown bias_dtype %d", what,
              bias_dtype);
  const int64_t ld_codes = round_up_to(k, 16);
  *used = codes ? 0 : round_up_to(rows * (ld_codes + 4), 16);
  FRX_REQUIRE(*used + more_bytes == 0 || (workspace != nullptr && aligned16(workspace) &&
                                          workspace_bytes >= *used + more_bytes),
              FRX_ERR_INVALID_ARG, "%s: workspace must be 16-byte aligned with %lld bytes (got %lld)", what,
              (long long)(*used + more_bytes), (long long)workspace_bytes);
  FRX_CHECK_RANGE(x, matrix_bytes(rows, k, ld_x, codes ? 1 : (x_dtype == FRX_DTYPE_F32 ? 4 : 2)), "int8 product: x");
  FRX_CHECK_RANGE(codes ? x_scale : nullptr, rows * 4, "int8 product: x_scale");
  FRX_CHECK_RANGE(w, matrix_bytes(cols, k, ld_w, 1), "int8 product: weight");
  FRX_CHECK_RANGE(w_scale, cols * 4, "int8 product: weight_scale");
  FRX_CHECK_RANGE(bias, cols * (bias_dtype == FRX_DTYPE_F32 ? 4 : 2), "int8 product: bias");
  FRX_CHECK_RANGE(workspace, *used + more_bytes, "int8 product: workspace");
  *op = {static_cast<const int8_t*>(x), ld_x, x_scale, w, ld_w, w_scale, bias, bias_dtype, rows, cols, k, !codes};
  if (!codes) {
    int8_t* c = static_cast<int8_t*>(workspace);
    float* sc = reinterpret_cast<float*>(c + rows * ld_codes);
    op->x = c;
    op->ld_x = ld_codes;
    op->x_scale = sc;
    return quantize(x, x_dtype, ld_x, rows, k, c, ld_codes, sc, stream);
  }
  return FRX_OK;
}

template <typename OutT>
static int launch_product(const I8Operands& op, void* out, int64_t ld_out, int* status, cudaStream_t stream) {
  I8Out p = {op.x_scale, op.w_scale, op.bias, op.bias_dtype, out, ld_out, static_cast<int>(op.rows),
             static_cast<int>(op.cols)};
  if (op.rows > kFewMaxTokens)
    return launch_gemm_i8<Int8StoreEpilogue<OutT>>(op.w, op.ld_w, op.x, op.ld_x, op.cols, op.rows, op.k, 16, p, status,
                                                   stream, op.quantised_here);
  const int nt = few_tokens_padded(op.rows);
  const int stages = few_stages(nt);
  CUtensorMap tm_w, tm_x;
  int rc = encode_8bit_2d(&tm_w, op.w, op.cols, op.k, op.ld_w, 128, 128);
  if (rc) return rc;
  rc = encode_8bit_2d(&tm_x, op.x, op.rows, op.k, op.ld_x, nt, 128);
  if (rc) return rc;
  static std::atomic<uint64_t> attr_done{0};
  auto kernel = gemm_i8_few_kernel<OutT>;
  constexpr int kMaxSmem = kFewRingBytes + 2048;
  rc = ensure_smem_attr(kernel, attr_done, kMaxSmem);
  if (rc) return rc;
  const int smem = stages * (kFewWBytes + nt * 128) + 2048;
  return launch_kernel(kernel, static_cast<unsigned>((op.cols + 127) / 128), kFewThreads, smem, stream,
                       op.quantised_here, tm_w, tm_x, p, nt, static_cast<int>((op.k + 127) / 128), stages, status);
}

template <bool kBias>
static int launch_score(const I8Operands& op, int64_t r0, int64_t n, const int64_t* target, float* partials,
                        int64_t tile_stride, int* status, cudaStream_t stream, bool overlap) {
  using Epi = Int8CEPartialsEpilogue<kBias>;
  typename Epi::Params ep;
  memset(&ep, 0, sizeof(ep));
  ep.row_scale = op.x_scale + r0;
  ep.col_scale = op.w_scale;
  ep.bias = op.bias;
  ep.bias_dtype = op.bias_dtype;
  ep.target = target + r0;
  ep.rows = static_cast<int>(n);
  ep.vocab_shard = static_cast<int>(op.cols);
  ep.partials = reinterpret_cast<float4*>(partials);
  ep.tile_stride = tile_stride;
  ep.n_tiles = static_cast<int>((op.cols + kBN - 1) / kBN);
  ep.status = status;
  return launch_gemm_i8<Epi>(op.x + r0 * op.ld_x, op.ld_x, op.w, op.ld_w, n, op.cols, op.k, 16, ep, status, stream,
                             overlap);
}

}  // namespace frx

extern "C" int frx_quantize_i8(const void* x, int dtype, int64_t ld_x, int64_t rows, int64_t cols, void* codes,
                               int64_t ld_codes, float* scale, void* stream) {
  using namespace frx;
  FRX_REQUIRE(rows >= 0 && cols >= 0 && ld_x >= cols && ld_codes >= cols && rows < (1ll << 31), FRX_ERR_INVALID_ARG,
              "frx_quantize_i8: bad sizes rows=%lld cols=%lld ld_x=%lld ld_codes=%lld", (long long)rows,
              (long long)cols, (long long)ld_x, (long long)ld_codes);
  FRX_REQUIRE(is_float_dtype(dtype), FRX_ERR_INVALID_ARG,
              "frx_quantize_i8: dtype must be FRX_DTYPE_BF16, FRX_DTYPE_F16 or FRX_DTYPE_F32");
  if (rows == 0) return FRX_OK;
  FRX_REQUIRE(scale != nullptr && (cols == 0 || (x != nullptr && codes != nullptr)), FRX_ERR_INVALID_ARG,
              "frx_quantize_i8: null pointer");
  FRX_CHECK_RANGE(x, matrix_bytes(rows, cols, ld_x, dtype == FRX_DTYPE_F32 ? 4 : 2), "frx_quantize_i8: x");
  FRX_CHECK_RANGE(codes, matrix_bytes(rows, cols, ld_codes, 1), "frx_quantize_i8: codes");
  FRX_CHECK_RANGE(scale, rows * 4, "frx_quantize_i8: scale");
  return quantize(x, dtype, ld_x, rows, cols, static_cast<int8_t*>(codes), ld_codes, scale,
                  static_cast<cudaStream_t>(stream));
}

extern "C" int frx_gemm_i8(const void* x, int x_dtype, int64_t ld_x, const float* x_scale, const void* weight,
                           int64_t ld_weight, const float* weight_scale, const void* bias, int bias_dtype,
                           int64_t rows, int64_t cols, int64_t k, void* workspace, int64_t workspace_bytes, void* out,
                           int64_t ld_out, int out_dtype, int* status, void* stream) {
  using namespace frx;
  FRX_REQUIRE(rows <= 0 || (out != nullptr && ld_out >= cols && is_float_dtype(out_dtype)), FRX_ERR_INVALID_ARG,
              "frx_gemm_i8: need an output with ld_out %lld >= cols %lld of dtype BF16, F16 or F32 (got %d)",
              (long long)ld_out, (long long)cols, out_dtype);
  if (rows > 0)
    FRX_CHECK_RANGE(out, matrix_bytes(rows, cols, ld_out, out_dtype == FRX_DTYPE_F32 ? 4 : 2), "frx_gemm_i8: out");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  I8Operands op;
  int64_t used = 0;
  const int rc = prepare_i8("frx_gemm_i8", x, x_dtype, ld_x, x_scale, weight, ld_weight, weight_scale, bias, bias_dtype,
                            rows, cols, k, workspace, workspace_bytes, &op, &used, 0, st);
  if (rc || rows == 0) return rc;
  if (out_dtype == FRX_DTYPE_F32) return launch_product<float>(op, out, ld_out, status, st);
  if (out_dtype == FRX_DTYPE_BF16) return launch_product<__nv_bfloat16>(op, out, ld_out, status, st);
  return launch_product<__half>(op, out, ld_out, status, st);
}

extern "C" int frx_i8_ce_entropy(const void* hidden, int hidden_dtype, int64_t ld_hidden, const float* hidden_scale,
                                 const void* weight, int64_t ld_weight, const float* weight_scale, const void* bias,
                                 int bias_dtype, const int64_t* target, int64_t rows, int64_t vocab_size,
                                 int64_t hidden_dim, int64_t ignore_index, int64_t launch_rows, void* workspace,
                                 int64_t workspace_bytes, float* ce, float* entropy, float* lse, float* log_probs,
                                 int* status, void* stream) {
  using namespace frx;
  FRX_REQUIRE(rows <= 0 || (launch_rows >= 1 && target != nullptr), FRX_ERR_INVALID_ARG,
              "frx_i8_ce_entropy: need targets and launch_rows >= 1 (got %lld)", (long long)launch_rows);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t n_tiles = vocab_size > 0 ? (vocab_size + kBN - 1) / kBN : 0;
  const int64_t step = launch_rows < rows ? launch_rows : rows;
  FRX_CHECK_RANGE(target, rows * 8, "frx_i8_ce_entropy: target");
  I8Operands op;
  int64_t used = 0;
  int rc = prepare_i8("frx_i8_ce_entropy", hidden, hidden_dtype, ld_hidden, hidden_scale, weight, ld_weight,
                      weight_scale, bias, bias_dtype, rows, vocab_size, hidden_dim, workspace, workspace_bytes, &op,
                      &used, rows > 0 ? n_tiles * step * 16 : 0, st);
  if (rc || rows == 0) return rc;
  float* partials = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + used);
  for (int64_t r0 = 0; r0 < rows; r0 += step) {
    const int64_t n = rows - r0 < step ? rows - r0 : step;
    const bool overlap = op.quantised_here && r0 == 0;
    rc = bias != nullptr ? launch_score<true>(op, r0, n, target, partials, step, status, st, overlap)
                         : launch_score<false>(op, r0, n, target, partials, step, status, st, overlap);
    if (rc) return rc;
    auto at = [r0](float* p) { return p == nullptr ? nullptr : p + r0; };
    rc = frx_finalize(partials, n_tiles, n, step, 0, target + r0, vocab_size, ignore_index, at(ce), at(entropy), at(lse),
                      at(log_probs), nullptr, status, stream);
    if (rc) return rc;
  }
  return FRX_OK;
}
