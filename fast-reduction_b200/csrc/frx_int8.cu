// The vocabulary head in 8-bit integers: hidden states quantised per token, times a weight whose
// rows (vocabulary entries) are 8-bit codes with one scale each.
//
//   frx_quantize_i8      scale_r = fl32(max_k |x_rk| / 127),  code_rk = nearest integer to
//                        x_rk / scale_r (ties to even)
//   frx_gemm_i8          y[r, j] = (sum_k code_rk w_jk) scale_r wscale_j + bias_j
//   frx_fwd_partials_i8  the same product reduced to softmax partials (m, s, u, zt) by the epilogue
//
// |code| <= 127, so a sum over K <= 131072 products stays below 2^31: the int32 accumulators of
// kind::i8 hold it exactly and the result does not depend on the order of the products.
#include <cstring>

#include "frx_epilogue.cuh"
#include "frx_host.cuh"

namespace frx {

constexpr int64_t kI8MaxK = 131072;

// ------------------------------------------------------------------------------------ quantisation
template <typename T>
struct Q8Vec;
template <>
struct Q8Vec<float> {
  __device__ static void load8(const float* p, float (&v)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p));
    const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  __device__ static float one(const float* p) { return __ldg(p); }
};
template <>
struct Q8Vec<__nv_bfloat16> {
  __device__ static void load8(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2(w[i], false);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  __device__ static float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
};
template <>
struct Q8Vec<__half> {
  __device__ static void load8(const __half* p, float (&v)[8]) {
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2(w[i], true);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  __device__ static float one(const __half* p) { return __half2float(*p); }
};

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

template <typename T>
__global__ void __launch_bounds__(kQ8Threads)
    quantize_i8_kernel(const T* __restrict__ x, int64_t ld_x, int64_t rows, int64_t cols, int8_t* __restrict__ codes,
                       int64_t ld_codes, float* __restrict__ scale_out, int vec_ok) {
  __shared__ float red[kQ8Threads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * ld_x;
    int8_t* cr = codes + row * ld_codes;
    const int64_t nv = vec_ok ? cols / 8 : 0;
    float amax = 0.0f;
    for (int64_t i = threadIdx.x; i < nv; i += kQ8Threads) {
      float v[8];
      Q8Vec<T>::load8(xr + 8 * i, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = amax_nan(amax, v[j]);
    }
    for (int64_t i = 8 * nv + threadIdx.x; i < cols; i += kQ8Threads) amax = amax_nan(amax, Q8Vec<T>::one(xr + i));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = amax_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (lane == 0) red[warp] = amax;
    __syncthreads();
    amax = red[0];
#pragma unroll
    for (int w = 1; w < kQ8Threads / 32; ++w) amax = amax_nan(amax, red[w]);
    float scale, inv;
    q8_scale(amax, scale, inv);
    if (threadIdx.x == 0) scale_out[row] = scale;
    const bool live = inv != 0.0f;
    for (int64_t i = threadIdx.x; i < nv; i += kQ8Threads) {
      float v[8];
      Q8Vec<T>::load8(xr + 8 * i, v);
      int k[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) k[j] = live ? q8_code(v[j], scale, inv) : 0;
      *reinterpret_cast<uint2*>(cr + 8 * i) =
          make_uint2(pack4_i8(k[0], k[1], k[2], k[3]), pack4_i8(k[4], k[5], k[6], k[7]));
    }
    for (int64_t i = 8 * nv + threadIdx.x; i < cols; i += kQ8Threads)
      cr[i] = static_cast<int8_t>(live ? q8_code(Q8Vec<T>::one(xr + i), scale, inv) : 0);
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------ epilogues
// One value of an optional bias vector (bf16, fp16 or fp32).
__device__ __forceinline__ float bias_at(const void* bias, int dtype, int64_t i) {
  if (dtype == FRX_DTYPE_F32) return __ldg(static_cast<const float*>(bias) + i);
  return unpack2(__ldg(static_cast<const uint16_t*>(bias) + i), dtype == FRX_DTYPE_F16).x;
}

// Output tile of the plain product. The weight is the A operand, so a thread owns one vocabulary entry
// (TMEM lane) and a warp's 32 lanes store 32 neighbouring outputs of one token: coalesced rows without
// staging, whatever the output's alignment.
struct Int8StoreEpilogue {
  static constexpr int kSmemPerWarp = 0;
  static constexpr int kSmemBytes = 0;

  struct Params {
    const float* row_scale;  // [rows] of the tokens
    const float* col_scale;  // [cols] of the weight's rows
    const void* bias;
    int bias_dtype;
    void* out;
    int64_t ld_out;
    int rows;
    int cols;
    int out_dtype;
  };

  template <class Release>
  __device__ __forceinline__ static void run(const Params& p, uint8_t* /*stage*/, uint32_t tacc, int m_blk, int n_blk,
                                             int q, int lane, Release release) {
    const int j = m_blk * kBM + q * 32 + lane;  // vocabulary entry
    const int r0 = n_blk * kBN;                 // first token
    const int ntok = min(kBN, p.rows - r0);
    const bool ok = j < p.cols;
    const float ws = ok ? __ldg(p.col_scale + j) : 0.0f;
    const float b = ok && p.bias != nullptr ? bias_at(p.bias, p.bias_dtype, j) : 0.0f;
    float v[32];
#pragma unroll 1
    for (int c = 0; c < kBN / 32; ++c) {
      const int lim = ntok - c * 32;
      if (lim <= 0) break;
      __syncwarp();
      tmem_load_32cols(tacc + static_cast<uint32_t>(c * 32), v);
      const float xs_lane = lane < lim ? __ldg(p.row_scale + r0 + c * 32 + lane) : 0.0f;
      const int64_t off = static_cast<int64_t>(r0 + c * 32) * p.ld_out + j;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float xs = __shfl_sync(0xffffffffu, xs_lane, i);
        const float y = static_cast<float>(__float_as_int(v[i])) * xs * ws + b;
        if (ok && i < lim) {
          const int64_t o = off + i * p.ld_out;
          if (p.out_dtype == FRX_DTYPE_F32)
            static_cast<float*>(p.out)[o] = y;
          else if (p.out_dtype == FRX_DTYPE_BF16)
            static_cast<__nv_bfloat16*>(p.out)[o] = __float2bfloat16_rn(y);
          else
            static_cast<__half*>(p.out)[o] = __float2half_rn(y);
        }
      }
    }
    release();
  }

  __device__ __forceinline__ static void finish(const Params&, int) {}
};

// Softmax partials of the scaled product: the two passes of the 16-bit forward's epilogue, with
// z = acc * row_scale * col_scale (+ bias) formed from the int32 accumulator in each pass.
struct Int8CEPartialsEpilogue {
  static constexpr int kSmemPerWarp = 0;
  static constexpr int kSmemBytes = 0;

  struct Params {
    const float* row_scale;
    const float* col_scale;
    const void* bias;
    int bias_dtype;
    int vec;  // col_scale (and an fp32 bias) 16-byte aligned
    const int64_t* target;
    int64_t vocab_offset;
    int rows;
    int vocab_shard;
    float4* partials;
    int64_t tile_stride;
    int n_tiles;
    int* status;
  };

  __device__ __forceinline__ static void dequant32(const Params& p, float (&v)[32], int col, int lim, float xs) {
    if (lim >= 32 && p.vec) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float4 s = __ldg(reinterpret_cast<const float4*>(p.col_scale + col) + k);
        const float f[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * k + i] = static_cast<float>(__float_as_int(v[4 * k + i])) * xs * f[i];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < lim) v[j] = static_cast<float>(__float_as_int(v[j])) * xs * __ldg(p.col_scale + col + j);
    }
    if (p.bias != nullptr) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < lim) v[j] += bias_at(p.bias, p.bias_dtype, col + j);
    }
  }

  template <class Release>
  __device__ __forceinline__ static void run(const Params& p, uint8_t* /*stage*/, uint32_t tacc, int m_blk, int n_blk,
                                             int q, int lane, Release release) {
    const int row = m_blk * kBM + q * 32 + lane;
    const int n0 = n_blk * kBN;
    const int ncols = min(kBN, p.vocab_shard - n0);
    const bool row_ok = row < p.rows;
    const float xs = row_ok ? __ldg(p.row_scale + row) : 0.0f;
    int tcol = -1;
    if (row_ok && p.target != nullptr) {
      const long long lt = static_cast<long long>(p.target[row]) - p.vocab_offset - n0;
      if (lt >= 0 && lt < ncols) tcol = static_cast<int>(lt);
    }
    float v[32];
    float mx = -INFINITY, zt = 0.0f;
#pragma unroll 1
    for (int c = 0; c < kBN / 32; ++c) {
      const int lim = ncols - c * 32;
      if (lim <= 0) break;
      __syncwarp();
      tmem_load_32cols(tacc + static_cast<uint32_t>(c * 32), v);
      dequant32(p, v, n0 + c * 32, lim, xs);
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j < lim) mx = fmaxf(mx, v[j]);
      if ((tcol >> 5) == c) zt = select32(v, tcol & 31);
    }
    float s0 = 0.f, s1 = 0.f, u0 = 0.f, u1 = 0.f;
#pragma unroll 1
    for (int c = 0; c < kBN / 32; ++c) {
      const int lim = ncols - c * 32;
      if (lim <= 0) break;
      __syncwarp();
      tmem_load_32cols(tacc + static_cast<uint32_t>(c * 32), v);
      dequant32(p, v, n0 + c * 32, lim, xs);
#pragma unroll
      for (int j = 0; j < 32; j += 2) {
        if (j < lim) {
          const float d = v[j] - mx;
          const float e = ex2_approx(d * kLog2e);
          s0 += e;
          u0 = fmaf(d, e, u0);
        }
        if (j + 1 < lim) {
          const float d = v[j + 1] - mx;
          const float e = ex2_approx(d * kLog2e);
          s1 += e;
          u1 = fmaf(d, e, u1);
        }
      }
    }
    release();
    if (row_ok && device_check(n_blk < p.n_tiles, p.status))
      p.partials[static_cast<int64_t>(n_blk) * p.tile_stride + row] = make_float4(mx, s0 + s1, u0 + u1, zt);
  }

  __device__ __forceinline__ static void finish(const Params&, int) {}
};

static bool is_float_dtype(int d) { return d == FRX_DTYPE_BF16 || d == FRX_DTYPE_F32 || d == FRX_DTYPE_F16; }

// Checks shared by the two products.
static int check_i8_operands(const char* what, const void* x, int64_t ld_x, const float* x_scale, const void* w,
                             int64_t ld_w, const float* w_scale, const void* bias, int bias_dtype, int64_t rows,
                             int64_t cols, int64_t k) {
  FRX_REQUIRE(rows >= 0 && cols >= 1 && k >= 1 && rows < (1ll << 31) && cols < (1ll << 31), FRX_ERR_INVALID_ARG,
              "%s: bad sizes rows=%lld cols=%lld k=%lld", what, (long long)rows, (long long)cols, (long long)k);
  FRX_REQUIRE(k <= kI8MaxK, FRX_ERR_UNSUPPORTED, "%s: k %lld > %lld could overflow the int32 accumulators", what,
              (long long)k, (long long)kI8MaxK);
  if (rows == 0) return FRX_OK;
  FRX_REQUIRE(x != nullptr && x_scale != nullptr && w != nullptr && w_scale != nullptr, FRX_ERR_INVALID_ARG,
              "%s: null codes or scale pointer", what);
  FRX_REQUIRE(aligned16(x) && aligned16(w) && ld_x % 16 == 0 && ld_w % 16 == 0 && ld_x >= k && ld_w >= k,
              FRX_ERR_INVALID_ARG,
              "%s: codes need 16-byte aligned bases and leading dimensions >= k that are multiples of 16 (got %lld, "
              "%lld)", what, (long long)ld_x, (long long)ld_w);
  FRX_REQUIRE(bias == nullptr || is_float_dtype(bias_dtype), FRX_ERR_INVALID_ARG, "%s: unknown bias_dtype %d", what,
              bias_dtype);
  FRX_CHECK_RANGE(x, matrix_bytes(rows, k, ld_x, 1), "int8 product: x");
  FRX_CHECK_RANGE(x_scale, rows * 4, "int8 product: x_scale");
  FRX_CHECK_RANGE(w, matrix_bytes(cols, k, ld_w, 1), "int8 product: weight");
  FRX_CHECK_RANGE(w_scale, cols * 4, "int8 product: weight_scale");
  FRX_CHECK_RANGE(bias, cols * (bias_dtype == FRX_DTYPE_F32 ? 4 : 2), "int8 product: bias");
  return FRX_OK;
}

template <typename T>
static int launch_quantize(const void* x, int64_t ld_x, int64_t rows, int64_t cols, int8_t* codes, int64_t ld_codes,
                           float* scale, cudaStream_t stream) {
  const int vec_ok = aligned16(x) && (ld_x * sizeof(T)) % 16 == 0 && (reinterpret_cast<uintptr_t>(codes) & 7u) == 0 &&
                     ld_codes % 8 == 0;
  const unsigned grid = static_cast<unsigned>(rows < (1 << 20) ? rows : (1 << 20));
  quantize_i8_kernel<T><<<grid, kQ8Threads, 0, stream>>>(static_cast<const T*>(x), ld_x, rows, cols, codes, ld_codes,
                                                         scale, vec_ok);
  FRX_CUDA_CHECK(cudaGetLastError());
  return FRX_OK;
}

}  // namespace frx

extern "C" int frx_quantize_i8(const void* x, int dtype, int64_t ld_x, int64_t rows, int64_t cols, void* codes,
                               int64_t ld_codes, float* scale, void* stream) {
  using namespace frx;
  FRX_REQUIRE(rows >= 0 && cols >= 0 && ld_x >= cols && ld_codes >= cols, FRX_ERR_INVALID_ARG,
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
  int8_t* c = static_cast<int8_t*>(codes);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == FRX_DTYPE_F32) return launch_quantize<float>(x, ld_x, rows, cols, c, ld_codes, scale, st);
  if (dtype == FRX_DTYPE_BF16) return launch_quantize<__nv_bfloat16>(x, ld_x, rows, cols, c, ld_codes, scale, st);
  return launch_quantize<__half>(x, ld_x, rows, cols, c, ld_codes, scale, st);
}

extern "C" int frx_gemm_i8(const void* x, int64_t ld_x, const float* x_scale, const void* weight, int64_t ld_weight,
                           const float* weight_scale, const void* bias, int bias_dtype, int64_t rows, int64_t cols,
                           int64_t k, void* out, int64_t ld_out, int out_dtype, int* status, void* stream) {
  using namespace frx;
  const int rc = check_i8_operands("frx_gemm_i8", x, ld_x, x_scale, weight, ld_weight, weight_scale, bias, bias_dtype,
                                   rows, cols, k);
  if (rc || rows == 0) return rc;
  FRX_REQUIRE(out != nullptr && ld_out >= cols && is_float_dtype(out_dtype), FRX_ERR_INVALID_ARG,
              "frx_gemm_i8: need an output with ld_out %lld >= cols %lld of dtype BF16, F16 or F32 (got %d)",
              (long long)ld_out, (long long)cols, out_dtype);
  FRX_CHECK_RANGE(out, matrix_bytes(rows, cols, ld_out, out_dtype == FRX_DTYPE_F32 ? 4 : 2), "frx_gemm_i8: out");
  Int8StoreEpilogue::Params ep;
  memset(&ep, 0, sizeof(ep));
  ep.row_scale = x_scale;
  ep.col_scale = weight_scale;
  ep.bias = bias;
  ep.bias_dtype = bias_dtype;
  ep.out = out;
  ep.ld_out = ld_out;
  ep.rows = static_cast<int>(rows);
  ep.cols = static_cast<int>(cols);
  ep.out_dtype = out_dtype;
  return launch_gemm_i8<Int8StoreEpilogue>(weight, ld_weight, x, ld_x, cols, rows, k, 16, ep, status,
                                           static_cast<cudaStream_t>(stream));
}

extern "C" int frx_fwd_partials_i8(const void* hidden, int64_t ld_hidden, const float* hidden_scale,
                                   const void* weight, int64_t ld_weight, const float* weight_scale, const void* bias,
                                   int bias_dtype, const int64_t* target, int64_t rows, int64_t vocab_shard,
                                   int64_t hidden_dim, int64_t vocab_offset, float* partials, int64_t tile_stride,
                                   int* status, void* stream) {
  using namespace frx;
  const int rc = check_i8_operands("frx_fwd_partials_i8", hidden, ld_hidden, hidden_scale, weight, ld_weight,
                                   weight_scale, bias, bias_dtype, rows, vocab_shard, hidden_dim);
  if (rc || rows == 0) return rc;
  FRX_REQUIRE(partials != nullptr && aligned16(partials) && tile_stride >= rows, FRX_ERR_INVALID_ARG,
              "frx_fwd_partials_i8: partials must be 16-byte aligned with tile_stride %lld >= rows %lld",
              (long long)tile_stride, (long long)rows);
  const int64_t n_tiles = (vocab_shard + kBN - 1) / kBN;
  FRX_CHECK_RANGE(target, rows * 8, "frx_fwd_partials_i8: target");
  FRX_CHECK_RANGE(partials, matrix_bytes(n_tiles, rows, tile_stride, 16), "frx_fwd_partials_i8: partials");
  Int8CEPartialsEpilogue::Params ep;
  memset(&ep, 0, sizeof(ep));
  ep.row_scale = hidden_scale;
  ep.col_scale = weight_scale;
  ep.bias = bias;
  ep.bias_dtype = bias_dtype;
  ep.vec = aligned16(weight_scale) ? 1 : 0;
  ep.target = target;
  ep.vocab_offset = vocab_offset;
  ep.rows = static_cast<int>(rows);
  ep.vocab_shard = static_cast<int>(vocab_shard);
  ep.partials = reinterpret_cast<float4*>(partials);
  ep.tile_stride = tile_stride;
  ep.n_tiles = static_cast<int>(n_tiles);
  ep.status = status;
  return launch_gemm_i8<Int8CEPartialsEpilogue>(hidden, ld_hidden, weight, ld_weight, rows, vocab_shard, hidden_dim, 16,
                                                ep, status, static_cast<cudaStream_t>(stream));
}
