// The vocabulary head in 8-bit integers: hidden states quantised per token, times a weight whose
// rows (vocabulary entries) are 8-bit codes with one scale each.
//
//   frx_quantize_i8      scale_r = fl32(max_k |x_rk| / 127),  code_rk = nearest integer to
//                        x_rk / scale_r (ties to even)
//   frx_gemm_i8          y[r, j] = (sum_k code_rk w_jk) scale_r wscale_j + bias_j
//   frx_i8_ce_entropy    the same product reduced to softmax partials (m, s, u, zt) by the epilogue, and
//                        those to cross-entropy, entropy and log-probability per row
//
// |code| <= 128, so a sum over K <= 131071 products stays below 2^31: the int32 accumulators of
// kind::i8 hold it exactly and the result does not depend on the order of the products.
//
// What bounds them (one B200; 6.56 TB/s is what a copy reaches):
//   quantisation    fp32 HBM: 128256 x 4096 364 us (7.2 TB/s); bf16 and fp16 issue slots (0.82 and 0.84 instructions per cycle
//                   and scheduler, HBM 52 %): 316 us (5.0 TB/s) and 275 us
//   few tokens      HBM: 1 token x 4096 x 128256 84 us (6.2 TB/s of weight), 64 tokens 92 us
//   many tokens     the tensor pipe's power and the L2's bandwidth to the SMs together: a 256 x 256 tile moves
//                   512 bytes per K and SM pair, 12 TB/s. 4096 tokens x 4096 x 32768 stored 418 us (2.6 POP/s),
//                   x 128256 scored 1.45 ms (3.0 POP/s, tensor pipe 91 % active at 1.55 GHz)
#include <cstring>
#include <type_traits>

#include "frx_epilogue.cuh"
#include "frx_host.cuh"

namespace frx {

constexpr int64_t kI8MaxK = FRX_I8_MAX_K;
static_assert(kI8MaxK * 128 * 128 < (1ll << 31) && (kI8MaxK + 1) * 128 * 128 >= (1ll << 31), "largest exact int32 sum");

// ------------------------------------------------------------------------------------ quantisation
// Eight consecutive values of a row as they lie in memory. max_bits folds the bits of |x| into a running
// maximum: as integers they order as the values do, with infinity and NaN above every finite one.
template <typename T>
struct Raw8 {  // 16-bit types; two maxima per word
  uint4 q;
  __device__ void load(const T* p) { q = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ uint32_t max_bits(uint32_t m) const {
    const uint32_t a = __vmaxu2(q.x & 0x7fff7fffu, q.y & 0x7fff7fffu);
    const uint32_t b = __vmaxu2(q.z & 0x7fff7fffu, q.w & 0x7fff7fffu);
    return __vmaxu2(m, __vmaxu2(a, b));
  }
  __device__ static uint32_t one_bits(const T* p) { return __ldg(reinterpret_cast<const uint16_t*>(p)) & 0x7fffu; }
  // the largest |x| of a folded word
  __device__ static float amax(uint32_t m) {
    return unpack2(max(m & 0xffffu, m >> 16), std::is_same<T, __half>::value).x;
  }
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
  uint4 a, b;
  __device__ void load(const float* p) {
    a = __ldg(reinterpret_cast<const uint4*>(p));
    b = __ldg(reinterpret_cast<const uint4*>(p) + 1);
  }
  __device__ uint32_t max_bits(uint32_t m) const {
    const uint32_t k = 0x7fffffffu;
    const uint32_t x = max(max(a.x & k, a.y & k), max(a.z & k, a.w & k));
    const uint32_t y = max(max(b.x & k, b.y & k), max(b.z & k, b.w & k));
    return max(m, max(x, y));
  }
  __device__ static uint32_t one_bits(const float* p) {
    return __ldg(reinterpret_cast<const uint32_t*>(p)) & 0x7fffffffu;
  }
  __device__ static float amax(uint32_t m) { return __uint_as_float(m); }
  __device__ void floats(float (&v)[8]) const {
    v[0] = __uint_as_float(a.x); v[1] = __uint_as_float(a.y); v[2] = __uint_as_float(a.z); v[3] = __uint_as_float(a.w);
    v[4] = __uint_as_float(b.x); v[5] = __uint_as_float(b.y); v[6] = __uint_as_float(b.z); v[7] = __uint_as_float(b.w);
  }
};

__device__ __forceinline__ float one_f32(const float* p) { return __ldg(p); }
__device__ __forceinline__ float one_f32(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float one_f32(const __half* p) { return __half2float(*p); }

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

// Nearest integers to the real quotients x / scale, ties to even, as 8-bit codes. y = x * inv is within
// 127 * 2^-22 of the quotient, so rounding y is right unless it lies within 1e-4 of a half; there the sign of
// x - half * scale, exact from one FMA, decides. Adding 1.5 * 2^23 rounds y and leaves its integer in the low
// bits of the sum: no conversion instructions, of which the GPU issues a quarter as many per clock.
constexpr float kRoundMagic = 12582912.0f;

__device__ __forceinline__ uint32_t code_at_half(float x, float y, float scale) {
  const float lo = floorf(y);
  const float r = fmaf(-(lo + 0.5f), scale, x);  // sign of x / scale - (lo + 1/2)
  const float even = 2.0f * rintf(0.5f * (lo + 0.5f));
  const float k = r > 0.0f ? lo + 1.0f : (r < 0.0f ? lo : even);
  return __float_as_uint(k + kRoundMagic);
}

// Rounded quotients as words whose low byte is the code; whether one of them lies next to a half.
template <int N>
__device__ __forceinline__ bool codes_of(const float (&v)[N], float inv, uint32_t (&k)[N]) {
  bool near_half = false;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float y = v[j] * inv;
    const float t = y + kRoundMagic;
    k[j] = __float_as_uint(t);
    near_half |= fabsf(y - (t - kRoundMagic)) > 0.4999f;
  }
  return near_half;
}

// The same where some quotient lies next to a half.
template <int N>
__device__ __forceinline__ void codes_at_halves(const float (&v)[N], float scale, float inv, uint32_t (&k)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float y = v[j] * inv;
    const float t = y + kRoundMagic;
    k[j] = fabsf(y - (t - kRoundMagic)) > 0.4999f ? code_at_half(v[j], y, scale) : __float_as_uint(t);
  }
}

// The low bytes of four words.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

constexpr int kQ8Threads = 128;
constexpr int kQ8Held = 4;

// A row belongs to kLanes threads (a warp, or the whole CTA). The row's first 32 * kLanes values stay in
// registers between the maximum and the codes, so such a row is read once, with all its loads in flight
// together; what is longer is read again. Vectors with a quotient next to a half are done a second time at the
// end, out of line: bf16 rows have one in most rows, and the code for it unrolled into the main path made that
// too long for the instruction cache (4096 rows of 4096: 23 us).
template <typename T, int kLanes>
__global__ void __launch_bounds__(kQ8Threads)
    quantize_i8_kernel(const T* __restrict__ x, int64_t ld_x, int64_t rows, int64_t cols, int8_t* __restrict__ codes,
                       int64_t ld_codes, float* __restrict__ scale_out, int vec_ok) {
  grid_dep_launch();
  __shared__ uint32_t red[kQ8Threads / 32];
  constexpr int kRows = kQ8Threads / kLanes;
  const int t = threadIdx.x % kLanes;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kLanes;
  if (kLanes == 32 && row >= rows) return;
  const T* xr = x + row * ld_x;
  int8_t* cr = codes + row * ld_codes;
  const int64_t nv = vec_ok ? cols / 8 : 0;
  Raw8<T> held[kQ8Held];
  uint32_t bits = 0;
#pragma unroll
  for (int h = 0; h < kQ8Held; ++h)
    if (t + h * kLanes < nv) held[h].load(xr + 8 * (t + h * kLanes));
#pragma unroll
  for (int h = 0; h < kQ8Held; ++h)
    if (t + h * kLanes < nv) bits = held[h].max_bits(bits);
  for (int64_t i = t + kQ8Held * kLanes; i < nv; i += kLanes) {
    Raw8<T> r;
    r.load(xr + 8 * i);
    bits = r.max_bits(bits);
  }
  float amax = Raw8<T>::amax(bits);
  bits = 0;
  for (int64_t i = 8 * nv + t; i < cols; i += kLanes) bits = max(bits, Raw8<T>::one_bits(xr + i));
  // as bits again, now of the fp32 value: NaN stays on top
  bits = max(__float_as_uint(amax), __float_as_uint(Raw8<T>::amax(bits)));
  bits = __reduce_max_sync(0xffffffffu, bits);
  if (kLanes > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = bits;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kQ8Threads / 32; ++w) bits = max(bits, red[w]);
  }
  amax = __uint_as_float(bits);
  float scale, inv;
  q8_scale(amax, scale, inv);
  if (t == 0) scale_out[row] = scale;
  const bool live = inv != 0.0f;
  auto store8 = [&](const uint32_t (&k)[8], int64_t i) {
    const uint2 c = make_uint2(low_bytes(k[0], k[1], k[2], k[3]), low_bytes(k[4], k[5], k[6], k[7]));
    *reinterpret_cast<uint2*>(cr + 8 * i) = live ? c : make_uint2(0, 0);
  };
  auto put8 = [&](const Raw8<T>& r, int64_t i) {
    float v[8];
    uint32_t k[8];
    r.floats(v);
    const bool near_half = codes_of<8>(v, inv, k);
    store8(k, i);
    return near_half;
  };
  uint64_t halves = 0;  // bit h: this thread's vector h (of the first 64) has a quotient next to a half
#pragma unroll
  for (int h = 0; h < kQ8Held; ++h)
    if (t + h * kLanes < nv && put8(held[h], t + h * kLanes)) halves |= 1ull << h;
  int64_t from = nv;  // later ones are all done again
#pragma unroll 1
  for (int64_t i = t + kQ8Held * kLanes, h = kQ8Held; i < nv; i += kLanes, ++h) {
    Raw8<T> r;
    r.load(xr + 8 * i);
    if (put8(r, i)) {
      if (h < 64)
        halves |= 1ull << h;
      else
        from = min(from, i);
    }
  }
#pragma unroll 1
  for (;;) {
    int64_t i;
    if (halves != 0) {
      i = t + static_cast<int64_t>(__ffsll(halves) - 1) * kLanes;
      halves &= halves - 1;
    } else if (from < nv) {
      i = from;
      from += kLanes;
    } else {
      break;
    }
    Raw8<T> r;
    r.load(xr + 8 * i);
    float v[8];
    uint32_t k[8];
    r.floats(v);
    codes_at_halves<8>(v, scale, inv, k);
    store8(k, i);
  }
#pragma unroll 1
  for (int64_t i = 8 * nv + t; i < cols; i += kLanes) {
    const float v[1] = {one_f32(xr + i)};
    uint32_t k[1];
    if (codes_of<1>(v, inv, k)) codes_at_halves<1>(v, scale, inv, k);
    cr[i] = static_cast<int8_t>(live ? k[0] & 0xffu : 0u);
  }
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
// coalesced rows without staging, whatever the output's alignment. s_scale: the tokens' 32 scales in shared
// memory, which every lane reads.
template <typename OutT>
__device__ __forceinline__ void store_tokens32(const I8Out& p, const float (&v)[32], const float* s_scale, int j, int r,
                                               float ws, float b) {
  const int lim = p.rows - r;
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
// vocabulary entry (TMEM lane); a warp has 128 of the tile's 256 tokens.
template <typename OutT>
struct Int8StoreEpilogue {
  static constexpr int kSmemBytes = 16 * 512;  // 128 scales per warp
  using Params = I8Out;

  struct Tile {
    float ws, b, xs[4];
  };

  __device__ __forceinline__ static Tile fetch(const Params& p, int m_blk, int n_blk, int half, int q, int lane) {
    const int j = m_blk * kBM + q * 32 + lane;
    const int r = n_blk * kBN + half * 128 + lane;
    const bool ok = j < p.cols;
    Tile t;
#pragma unroll
    for (int i = 0; i < 4; ++i) t.xs[i] = r + i * 32 < p.rows ? ld_dep_f32(p.row_scale + r + i * 32) : 0.0f;
    t.ws = ok ? __ldg(p.col_scale + j) : 0.0f;
    t.b = ok && p.bias != nullptr ? bias_at(p.bias, p.bias_dtype, j) : 0.0f;
    return t;
  }

  __device__ __forceinline__ static void stage(const Tile& t, uint8_t* smem, int group, int half, int q, int lane) {
    float* s_scale = reinterpret_cast<float*>(smem) + ((group * 2 + half) * 4 + q) * 128;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) s_scale[i * 32 + lane] = t.xs[i];
    __syncwarp();
  }

  template <class Release, class Wait>
  __device__ __forceinline__ static bool run(const Params& p, const Tile& tile, uint8_t* smem, uint32_t tacc, int m_blk,
                                             int n_blk, int group, int half, int q, int lane, uint64_t* /*join*/,
                                             uint32_t& /*joins*/, Release release, Wait /*wait*/) {
    const int j = m_blk * kBM + q * 32 + lane;  // vocabulary entry
    const int r0 = n_blk * kBN + half * 128;    // first token
    const int ntok = min(128, p.rows - r0);
    const float* s_scale = reinterpret_cast<float*>(smem) + ((group * 2 + half) * 4 + q) * 128;
    if (j - lane < p.cols) {
      float v[32];
#pragma unroll 1
      for (int c = 0; c < ntok; c += 32) {
        __syncwarp();
        tmem_load_32cols(tacc + static_cast<uint32_t>(c), v);
        store_tokens32<OutT>(p, v, s_scale + c, j, r0 + c, tile.ws, tile.b);
      }
    }
    release();
    return true;
  }

  __device__ __forceinline__ static void finish(const Params&, int) {}
};

constexpr float kLow = -1e38f;  // below every logit; differences to it stay finite

// The partial of columns none of which is live: empty, or NaN when the sum says that one of them is NaN (maxima drop
// it, and the merge skips a maximum of -inf).
__device__ __forceinline__ float4 nothing_live(float s, float zt) {
  return s == s ? make_float4(-INFINITY, 0.0f, 0.0f, zt) : make_float4(s, s, s, zt);
}

// Softmax partials of the scaled product, in one pass over the accumulator: thread = token (TMEM lane), 16
// columns at a time with a running maximum, and s and u rescaled when it rises. A warp has 128 of the tile's
// 256 columns; the two warps of a token join their statistics through shared memory. Pairs of columns share
// fp32x2 instructions: a pair costs two int32 conversions, two exponentials, two maxima and five others.
//   kFull = false: the token's scale xs >= 0 is taken out: with y = acc * wscale, z = xs y has its maximum where
//     y has, exp(z - m) = 2^((y - max y) xs log2 e), u = xs sum (y - max y) e.
//   kFull = true: z = (acc * wscale) * xs + bias, for a bias and for the caller's own scales (any sign).
template <bool kFull>
struct Int8CEPartialsEpilogue {
  static constexpr int kJoinBytes = 2 * 8 * 32 * 16;  // (receiving half, group, quarter) x 32 tokens
  static constexpr int kSmemBytes = kJoinBytes + 16 * 1024;  // and 128 scales and 128 biases per warp

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

  struct Tile {
    float xs, ws[4], b[kFull ? 4 : 1];
    int tcol;  // the target's column among this warp's 128, if it is one of them
  };

  __device__ __forceinline__ static float* scales(uint8_t* smem, int group, int half, int q) {
    return reinterpret_cast<float*>(smem + kJoinBytes) + ((group * 2 + half) * 4 + q) * 256;
  }

  __device__ __forceinline__ static Tile fetch(const Params& p, int m_blk, int n_blk, int half, int q, int lane) {
    const int row = m_blk * kBM + q * 32 + lane;
    const int n0 = n_blk * kBN + half * 128;
    Tile t{};
    t.tcol = -1;
    if (row - lane >= p.rows) return t;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = n0 + i * 32 + lane;
      t.ws[i] = col < p.vocab_shard ? __ldg(p.col_scale + col) : 0.0f;
      if (kFull) t.b[i] = col < p.vocab_shard && p.bias != nullptr ? bias_at(p.bias, p.bias_dtype, col) : 0.0f;
    }
    if (row < p.rows) {
      t.xs = ld_dep_f32(p.row_scale + row);
      const int64_t lt = p.target[row] - n0;
      t.tcol = lt >= 0 && lt < min(128, p.vocab_shard - n0) ? static_cast<int>(lt) : -1;
    }
    return t;
  }

  __device__ __forceinline__ static void stage(const Tile& t, uint8_t* smem, int group, int half, int q, int lane) {
    float* s_ws = scales(smem, group, half, q);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s_ws[i * 32 + lane] = t.ws[i];
      if (kFull) s_ws[128 + i * 32 + lane] = t.b[i];
    }
    __syncwarp();
  }

  struct Stat {
    float m, s, u, zt;
  };

  // 16 columns: r are their sums, s_ws their scales (and biases 128 behind them), `lim` of them valid; tcol the
  // target's column among them, or -1.
  template <bool kRagged>
  __device__ __forceinline__ static void columns16(Stat& st, const uint32_t (&r)[16], const float* s_ws, int lim,
                                                   uint64_t xs2, float k, uint64_t k2, int tcol) {
    uint64_t y[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(s_ws + 4 * i);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int j = 4 * i + 2 * h;
        y[2 * i + h] = mul_f32x2(pack_f32x2(static_cast<float>(static_cast<int>(r[j])),
                                            static_cast<float>(static_cast<int>(r[j + 1]))), h == 0 ? w.x : w.y);
      }
      if (kFull) {
        const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(s_ws + 128 + 4 * i);
        y[2 * i] = fma_f32x2(y[2 * i], xs2, b.x);
        y[2 * i + 1] = fma_f32x2(y[2 * i + 1], xs2, b.y);
      }
    }
    float v[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) unpack_f32x2(y[i], v[2 * i], v[2 * i + 1]);
    if (kRagged) {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (j >= lim) v[j] = kLow;
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = pack_f32x2(v[2 * i], v[2 * i + 1]);
    }
    if (tcol >= 0) st.zt = select16(v, tcol);
    if (kFull) {  // a bias of -inf masks its column: kLow contributes nothing, and -inf times 0 would be NaN
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = v[j] < kLow ? kLow : v[j];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = pack_f32x2(v[2 * i], v[2 * i + 1]);
    }
    float t4[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) t4[q] = fmaxf(fmaxf(v[4 * q], v[4 * q + 1]), fmaxf(v[4 * q + 2], v[4 * q + 3]));
    const float top = fmaxf(st.m, fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])));
    const float d = st.m - top;
    const float e0 = ex2_approx(d * k);
    const uint64_t neg = pack_f32x2(-top, -top);
    uint64_t s2[2] = {0, 0}, u2[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint64_t dd = add_f32x2(y[i], neg);
      float a0, a1;
      unpack_f32x2(mul_f32x2(dd, k2), a0, a1);
      a0 = ex2_approx(a0);
      a1 = ex2_approx(a1);
      if (kRagged) {
        a0 = 2 * i < lim ? a0 : 0.0f;
        a1 = 2 * i + 1 < lim ? a1 : 0.0f;
      }
      const uint64_t e = pack_f32x2(a0, a1);
      s2[i & 1] = add_f32x2(s2[i & 1], e);
      u2[i & 1] = fma_f32x2(dd, e, u2[i & 1]);
    }
    // s * e0 first: columns behind a mask (or with logits of -1e37) leave a d whose product with s passes the
    // largest float, and infinity times an e0 of 0 would be NaN
    st.s *= e0;
    st.u = fmaf(d, st.s, st.u * e0);
    st.m = top;
    float f0, f1;
    unpack_f32x2(add_f32x2(s2[0], s2[1]), f0, f1);
    st.s += f0 + f1;
    unpack_f32x2(add_f32x2(u2[0], u2[1]), f0, f1);
    st.u += f0 + f1;
  }

  template <class Release, class Wait>
  __device__ __forceinline__ static bool run(const Params& p, const Tile& tile, uint8_t* smem, uint32_t tacc, int m_blk,
                                             int n_blk, int group, int half, int q, int lane, uint64_t* join,
                                             uint32_t& joins, Release release, Wait wait) {
    const int row0 = m_blk * kBM + q * 32;
    const int row = row0 + lane;
    if (row0 >= p.rows) {  // both warps of these tokens
      release();
      return true;
    }
    const int n0 = n_blk * kBN + half * 128;
    const int ncols = min(128, p.vocab_shard - n0);
    const bool row_ok = row < p.rows;
    const float* s_ws = scales(smem, group, half, q);
    const float xs = tile.xs;
    const float k = kFull ? kLog2e : xs * kLog2e;
    const uint64_t k2 = pack_f32x2(k, k), xs2 = pack_f32x2(xs, xs);
    const int tcol = tile.tcol;
    Stat st = {kLow, 0.0f, 0.0f, 0.0f};
    uint32_t r[16];
    if (ncols == 128) {
#pragma unroll 1
      for (int c = 0; c < 128; c += 16) {
        __syncwarp();
        tmem_load_16cols(tacc + static_cast<uint32_t>(c), r);
        columns16<false>(st, r, s_ws + c, 16, xs2, k, k2, (tcol >> 4) == (c >> 4) ? tcol & 15 : -1);
      }
    } else {
#pragma unroll 1
      for (int c = 0; c < ncols; c += 16) {
        __syncwarp();
        tmem_load_16cols(tacc + static_cast<uint32_t>(c), r);
        columns16<true>(st, r, s_ws + c, ncols - c, xs2, k, k2, (tcol >> 4) == (c >> 4) ? tcol & 15 : -1);
      }
    }
    if (kFull && st.m <= kLow) {
      const float4 n = nothing_live(st.s, st.zt);
      st = {n.x, n.y, n.z, n.w};
    }
    const float f = kFull ? 1.0f : xs;
    st.m *= f;
    st.u *= f;
    st.zt *= f;
    // One half hands its statistics to the other through shared memory, in turn: the first half receives the pair's first
    // tile's, the second half the next one's. A half that writes its slot has then received since the other read it (its
    // own wait on the other's arrival, which follows that read), so no write passes a read.
    const int turn = static_cast<int>(joins & 1u);
    const uint32_t parity = (joins >> 1) & 1u;
    ++joins;
    float4* slot = reinterpret_cast<float4*>(smem) + ((turn * 2 + group) * 4 + q) * 32 + lane;
    if (half != turn) {
      *slot = make_float4(st.m, st.s, st.u, st.zt);
      __syncwarp();
      if (lane == 0) mbar_arrive(join + turn);
      release();
      return true;
    }
    if (!wait(join + turn, parity)) return false;
    const float4 o = *slot;
    release();
    st.zt += o.w;
    if (st.s == 0.0f) {  // nothing in this half
      st = {o.x, o.y, o.z, st.zt};
    } else if (o.y != 0.0f) {  // something in the other one (the tile need not reach the second)
      const float top = fmaxf(st.m, o.x);
      const float d0 = st.m - top, d1 = o.x - top;
      const float e0 = ex2_approx(d0 * kLog2e), e1 = ex2_approx(d1 * kLog2e);
      const float s0 = st.s * e0, s1 = o.y * e1;
      st.u = fmaf(d0, s0, st.u * e0) + fmaf(d1, s1, o.z * e1);  // as in columns16
      st.s = s0 + s1;
      st.m = top;
    }
    if (row_ok && device_check(n_blk < p.n_tiles, p.status))
      p.partials[static_cast<int64_t>(n_blk) * p.tile_stride + row] = make_float4(st.m, st.s, st.u, st.zt);
    return true;
  }

  __device__ __forceinline__ static void finish(const Params&, int) {}
};

// ------------------------------------------------------------------------------------ few tokens
// Up to 128 tokens: the product streams the weight once and is bound by HBM. The vocabulary is the M of the MMA and
// the tokens are its N (rounded up to 16), so the tokens' padding costs nothing in HBM. Two persistent CTAs per SM
// walk tiles of 128 vocabulary entries: warp 0 keeps the ring of 128-byte deep K steps filled across tiles, warp 1
// issues the MMAs, and four warps drain the finished one of two accumulators, so neither a tile's start nor its
// end interrupts the stream (64 tokens x 4096 x 128256: 102 -> 96 us; one CTA per SM on 256 entries, which reads the
// tokens half as often, took 99). The first ring of weight tiles is requested before the wait for the tokens'
// quantisation. The ring holds at most 4 steps, 128 KB of weight in flight per SM (1 token: 88.7 us with 6 steps, 84.1
// with 4, 86 with 3, 97 with 2), and the weight is marked to leave the L2 first, so that the tokens stay
// (64 tokens: 96 -> 92 us).
// Against the CTA-pair core, us at 4096 x 128256 and 1024 x 32000, bf16 in and out, inputs larger than the L2 (its loads of
// token rows that do not exist are slow):
//   storing   1 token 83 : 132, 11 : 16    64 tokens 87 : 98, 12 : 16      128 tokens 95 : 106, 15 : 16
//   scoring   1 token 94 : 140, 17 : 21    64 tokens 98 : 105, 20 : 22     128 tokens 124 : 109, 28 : 20
constexpr int kFewMaxTokens = 128;
constexpr int kFewMaxScored = FRX_I8_FEW_ROWS;
constexpr int kFewWBytes = 128 * 128;
constexpr int kFewThreads = 192;
constexpr int kFewSmemBudget = 115712;  // of 228 KiB per SM for two CTAs, each with 1 KiB for the system
constexpr int kFewMaxStages = 4;

inline int few_tokens_padded(int64_t rows) { return static_cast<int>((rows + 15) / 16 * 16); }

// What an epilogue warp works with: entries 32 q .. 32 q + 31 of a tile.
struct FewWarp {
  int tile;
  int buf;  // accumulator
  int q, lane;
  uint32_t tacc;
  float ws, b;  // scale and bias of this lane's entry
  const float* s_scale;
};

// Stores the product.
template <typename OutT>
struct FewStore {
  using Params = I8Out;
  static constexpr int kSmemBytes = 0;
  __device__ __forceinline__ static const I8Out& operands(const Params& p) { return p; }
  __device__ __forceinline__ static void init(const Params&, uint8_t*, int) {}

  template <class Release, class Wait>
  __device__ __forceinline__ static bool run(const Params& p, const FewWarp& w, uint8_t* /*smem*/, uint64_t* /*join*/,
                                             uint32_t /*parity*/, int* /*status*/, Release release, Wait /*wait*/) {
    const int j = w.tile * 128 + w.q * 32 + w.lane;
    if (j - w.lane < p.cols) {
      float v[32];
#pragma unroll 1
      for (int c = 0; c < p.rows; c += 32) {
        __syncwarp();
        tmem_load_32cols(w.tacc + static_cast<uint32_t>(c), v);
        store_tokens32<OutT>(p, v, w.s_scale + c, j, c, w.ws, w.b);
      }
    }
    release();
    return true;
  }
};

// After it, lane i holds the reduction of a[i] over the warp's lanes: at each step a lane keeps the half of its values
// that its number points to and gives the other half away (31 shuffles instead of 160).
template <class Op>
__device__ __forceinline__ float reduce_transposed(float (&a)[32], int lane, Op op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (i < o) {
        const float keep = up ? a[i + o] : a[i], give = up ? a[i] : a[i + o];
        a[i] = op(keep, __shfl_xor_sync(0xffffffffu, give, o));
      }
    }
  }
  return a[0];
}

// Reduces the product to softmax partials of 128 columns. A warp reduces its 32 columns for 32 tokens at a time, lane =
// token after reduce_transposed; the first warp joins the four.
struct FewScore {
  struct Params {
    I8Out op;  // no output
    const int64_t* target;
    float4* partials;
    int64_t tile_stride;
    int n_tiles;
  };
  // joins: [accumulator][warps 1 to 3][token]; targets' logits: [warp][token]; targets
  static constexpr int kJoinBytes = 2 * 3 * kFewMaxScored * 16;
  static constexpr int kZtBytes = 4 * kFewMaxScored * 4;
  static constexpr int kSmemBytes = kJoinBytes + kZtBytes + kFewMaxScored * 4;
  __device__ __forceinline__ static const I8Out& operands(const Params& p) { return p.op; }

  // The targets as 32-bit ids (-1: not one of the vocabulary's).
  __device__ __forceinline__ static void init(const Params& p, uint8_t* smem, int thread) {
    int* s_target = reinterpret_cast<int*>(smem + kJoinBytes + kZtBytes);
    if (thread < kFewMaxScored) {
      const int64_t t = thread < p.op.rows ? p.target[thread] : -1;
      s_target[thread] = t >= 0 && t < p.op.cols ? static_cast<int>(t) : -1;
    }
  }

  template <class Release, class Wait>
  __device__ __forceinline__ static bool run(const Params& p, const FewWarp& w, uint8_t* smem, uint64_t* join,
                                             uint32_t parity, int* status, Release release, Wait wait) {
    const int rows = p.op.rows, lane = w.lane;
    const int j = w.tile * 128 + w.q * 32 + lane;
    const bool live = j < p.op.cols;
    float4* slots = reinterpret_cast<float4*>(smem) + w.buf * 3 * kFewMaxScored;
    float* s_zt = reinterpret_cast<float*>(smem + kJoinBytes) + w.q * kFewMaxScored;
    const int* s_target = reinterpret_cast<const int*>(smem + kJoinBytes + kZtBytes);
    float4 own[kFewMaxScored / 32];
    auto max2 = [](float x, float y) { return fmaxf(x, y); };
    auto add2 = [](float x, float y) { return x + y; };
#pragma unroll
    for (int g = 0; g < kFewMaxScored / 32; ++g) {
      const int c = g * 32;
      if (c < rows) {
        float v[32], a[32];
        __syncwarp();
        s_zt[c + lane] = 0.0f;
        __syncwarp();
        tmem_load_32cols(w.tacc + static_cast<uint32_t>(c), v);
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          v[i] = fmaf(static_cast<float>(__float_as_int(v[i])) * w.s_scale[c + i], w.ws, w.b);
          if (s_target[c + i] == j) s_zt[c + i] = v[i];
          v[i] = v[i] < kLow ? kLow : v[i];  // a bias of -inf masks its column
          a[i] = live ? v[i] : -INFINITY;
        }
        const float m = reduce_transposed(a, lane, max2);
        float u[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float d = v[i] - __shfl_sync(0xffffffffu, m, i);
          const float e = ex2_approx(d * kLog2e);
          a[i] = live ? e : 0.0f;
          u[i] = live ? d * e : 0.0f;
        }
        const float s = reduce_transposed(a, lane, add2);
        const float us = reduce_transposed(u, lane, add2);
        __syncwarp();
        own[g] = make_float4(m, s, us, s_zt[c + lane]);
        if (m <= kLow) own[g] = nothing_live(s, own[g].w);
        if (w.q != 0) slots[(w.q - 1) * kFewMaxScored + c + lane] = own[g];
      }
    }
    if (w.q != 0) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&join[w.buf]);
      release();
      return true;
    }
    // the others write these slots again only for the accumulator's next tile, which waits for this release
    if (!wait(&join[w.buf], parity)) return false;
#pragma unroll
    for (int g = 0; g < kFewMaxScored / 32; ++g) {
      const int token = g * 32 + lane;
      if (g * 32 < rows) {
        float4 t = own[g];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          const float4 o = slots[k * kFewMaxScored + token];
          t.w += o.w;
          if (o.y == 0.0f) continue;  // nothing there
          if (t.y == 0.0f) {
            t = make_float4(o.x, o.y, o.z, t.w);
            continue;
          }
          const float top = fmaxf(t.x, o.x);
          const float d0 = t.x - top, d1 = o.x - top;
          const float e0 = ex2_approx(d0 * kLog2e), e1 = ex2_approx(d1 * kLog2e);
          const float s0 = t.y * e0, s1 = o.y * e1;
          t.z = fmaf(d0, s0, t.z * e0) + fmaf(d1, s1, o.z * e1);  // as in columns16
          t.y = s0 + s1;
          t.x = top;
        }
        if (token < rows && w.tile * 128 < p.op.cols && device_check(w.tile < p.n_tiles, status))
          p.partials[w.tile * p.tile_stride + token] = t;
      }
    }
    release();
    return true;
  }
};

template <class Epi>
__global__ void __launch_bounds__(kFewThreads, 2)
    gemm_i8_few_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                       const __grid_constant__ typename Epi::Params ep, int nt, int num_k, int stages, int num_tiles,
                       int* status) {
  const I8Out& p = Epi::operands(ep);
  grid_dep_launch();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int w_bytes = kFewWBytes;
  const int x_bytes = nt * 128;
  uint8_t* s_w = smem;
  uint8_t* s_x = smem + stages * w_bytes;
  float* s_scale = reinterpret_cast<float*>(s_x + stages * x_bytes);  // the tokens', per epilogue warp
  uint8_t* s_epi = reinterpret_cast<uint8_t*>(s_scale + 4 * kFewMaxTokens);
  uint64_t* full = reinterpret_cast<uint64_t*>(s_epi + Epi::kSmemBytes);
  uint64_t* empty = full + kFewMaxStages;
  uint64_t* acc_full = empty + kFewMaxStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* join = acc_empty + 2;  // per accumulator
  uint64_t* done = join + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  if (!device_check(reinterpret_cast<const uint8_t*>(tmem_slot + 2) - smem_raw <=
                        static_cast<ptrdiff_t>(dynamic_smem_bytes()),
                    threadIdx.x == 0 ? status : nullptr))
    return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t acc_cols = nt <= 32 ? 32u : (nt <= 64 ? 64u : 128u);
  const uint32_t tmem_cols = 2 * acc_cols;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 4);
      mbar_init(&join[b], 3);
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
  if (warp >= 2) Epi::init(ep, s_epi, threadIdx.x - 64);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int my_tiles = (num_tiles - static_cast<int>(blockIdx.x) + static_cast<int>(gridDim.x) - 1) /
                       static_cast<int>(gridDim.x);  // tiles blockIdx.x, blockIdx.x + gridDim.x, ...

  if (warp == 0) {
    if (lane == 0) {
      const long long total = static_cast<long long>(my_tiles) * num_k;
      const int pre = static_cast<int>(total < stages ? total : stages);
      // K steps in order, over all tiles: w and x are asked for in step `it` of stage it % stages
      int tile = static_cast<int>(blockIdx.x), kb = 0;
      const uint64_t once = l2_evict_first();  // the weight; the tokens stay in the L2
      auto load_w = [&](int stage) {
        mbar_arrive_expect_tx(&full[stage], static_cast<uint32_t>(w_bytes + x_bytes));
        tma_load_2d_hint(s_w + stage * w_bytes, &tm_w, &full[stage], kb * 128, tile * 128, once);
      };
      auto next_step = [&]() {
        if (++kb == num_k) {
          kb = 0;
          tile += static_cast<int>(gridDim.x);
        }
      };
      for (int s = 0; s < pre; ++s, next_step()) load_w(s);
      grid_dep_wait();
      for (int s = 0; s < pre; ++s) tma_load_2d(s_x + s * x_bytes, &tm_x, &full[s], (s % num_k) * 128, 0);
      int stage = 0;
      uint32_t phase = 0;  // of empty[stage] to wait for
      long long it = pre;
      for (; it < total; ++it, next_step()) {
        if (!mbar_wait_bounded(&empty[stage], phase, abort_flag, status, kStatusTimeoutProducer))
          break;
        load_w(stage);
        tma_load_2d(s_x + stage * x_bytes, &tm_x, &full[stage], kb * 128, 0);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (it < total) {
        // gave up: let every copy still in flight land before the shared memory goes away
        for (long long i = it > stages ? it - stages : 0; i < it; ++i)
          mbar_wait_drain(&full[i % stages], static_cast<uint32_t>((i / stages) & 1), status);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = make_idesc_i8(128, nt);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int i = 0; i < my_tiles && ok; ++i) {
        const int buf = i & 1;
        if (!mbar_wait_bounded(&acc_empty[buf], static_cast<uint32_t>((i >> 1) & 1) ^ 1u, abort_flag, status,
                               kStatusTimeoutMma))
          break;
        tc_fence_after();
        for (int kb = 0; kb < num_k; ++kb) {
          if (!mbar_wait_bounded(&full[stage], phase, abort_flag, status, kStatusTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t w_addr = smem_u32(s_w + stage * w_bytes);
          const uint32_t x_addr = smem_u32(s_x + stage * x_bytes);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_i8(tmem + buf * acc_cols, make_smem_desc_sw128(w_addr + k * 32, 16, 1024),
                    make_smem_desc_sw128(x_addr + k * 32, 16, 1024), idesc, (kb | k) != 0 ? 1u : 0u);
          umma_commit(&empty[stage]);
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok) umma_commit(&acc_full[buf]);
      }
      umma_commit(done);
      mbar_wait_drain(done, 0, status);  // before TMEM is released
    }
    __syncwarp();
  } else {
    FewWarp w;
    w.q = warp & 3;
    w.lane = lane;
    auto entry = [&](int i, float& ws, float& b) {  // of the i-th tile
      const int tile = static_cast<int>(blockIdx.x) + i * static_cast<int>(gridDim.x);
      const int j = tile * 128 + w.q * 32 + lane;
      const bool ok = j < p.cols;
      ws = ok ? __ldg(p.col_scale + j) : 0.0f;
      b = ok && p.bias != nullptr ? bias_at(p.bias, p.bias_dtype, j) : 0.0f;
    };
    float ws = 0.0f, b = 0.0f;
    entry(0, ws, b);
    grid_dep_wait();
    float* s = s_scale + w.q * kFewMaxTokens;
#pragma unroll
    for (int i = 0; i < kFewMaxTokens; i += 32)
      if (i < p.rows) s[i + lane] = i + lane < p.rows ? ld_dep_f32(p.row_scale + i + lane) : 0.0f;
    __syncwarp();
    w.s_scale = s;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      int good = 1;
      if (lane == 0)
        good = mbar_wait_bounded(bar, parity, abort_flag, status, kStatusTimeoutEpilogue);
      return __shfl_sync(0xffffffffu, good, 0) != 0;
    };
    auto join_wait = [&](uint64_t* bar, uint32_t parity) {
      // by every lane, since what the barrier hands over is every lane's to read
      return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag, status, kStatusTimeoutEpilogue)) != 0;
    };
    for (int i = 0; i < my_tiles; ++i) {
      w.buf = i & 1;
      const uint32_t parity = static_cast<uint32_t>((i >> 1) & 1);
      w.ws = ws;
      w.b = b;
      if (i + 1 < my_tiles) entry(i + 1, ws, b);  // requested under this tile
      if (!wait(&acc_full[w.buf], parity)) break;
      tc_fence_after();
      w.tile = static_cast<int>(blockIdx.x) + i * static_cast<int>(gridDim.x);
      w.tacc = tmem + w.buf * acc_cols + (static_cast<uint32_t>(w.q * 32) << 16);
      auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[w.buf]);
      };
      if (!Epi::run(ep, w, s_epi, join, parity, status, release, join_wait)) break;
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

// Rows of up to 1024 values, which a warp holds in registers, go to a warp each (16384 rows of 1024 bf16: 15 us, with
// a CTA per row 24), longer ones to a CTA (a warp would read them twice).
template <typename T>
static int launch_quantize(const void* x, int64_t ld_x, int64_t rows, int64_t cols, int8_t* codes, int64_t ld_codes,
                           float* scale, cudaStream_t stream) {
  const int vec_ok = aligned16(x) && (ld_x * sizeof(T)) % 16 == 0 && (reinterpret_cast<uintptr_t>(codes) & 7u) == 0 &&
                     ld_codes % 8 == 0;
  const T* xt = static_cast<const T*>(x);
  if (cols <= 32 * 8 * kQ8Held) {
    constexpr int kRows = kQ8Threads / 32;
    quantize_i8_kernel<T, 32><<<static_cast<unsigned>((rows + kRows - 1) / kRows), kQ8Threads, 0, stream>>>(
        xt, ld_x, rows, cols, codes, ld_codes, scale, vec_ok);
  } else {
    quantize_i8_kernel<T, kQ8Threads><<<static_cast<unsigned>(rows), kQ8Threads, 0, stream>>>(
        xt, ld_x, rows, cols, codes, ld_codes, scale, vec_ok);
  }
  FRX_CUDA_CHECK(cudaGetLastError());
  return FRX_OK;
}

static int quantize(const void* x, int dtype, int64_t ld_x, int64_t rows, int64_t cols, int8_t* codes,
                    int64_t ld_codes, float* scale, cudaStream_t stream) {
  if (dtype == FRX_DTYPE_F32) return launch_quantize<float>(x, ld_x, rows, cols, codes, ld_codes, scale, stream);
  if (dtype == FRX_DTYPE_BF16)
    return launch_quantize<__nv_bfloat16>(x, ld_x, rows, cols, codes, ld_codes, scale, stream);
  return launch_quantize<__half>(x, ld_x, rows, cols, codes, ld_codes, scale, stream);
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

template <class Epi>
static int launch_few(const I8Operands& op, const typename Epi::Params& ep, int* status, cudaStream_t stream) {
  const int nt = few_tokens_padded(op.rows);
  // alignment, the tokens' scales, the epilogue's, barriers
  constexpr int kOther = 1024 + 4 * kFewMaxTokens * 4 + Epi::kSmemBytes + 256;
  const int stage_bytes = kFewWBytes + nt * 128;
  const int fit = (kFewSmemBudget - kOther) / stage_bytes;
  const int stages = fit < kFewMaxStages ? fit : kFewMaxStages;
  CUtensorMap tm_w, tm_x;
  int rc = encode_8bit_2d(&tm_w, op.w, op.cols, op.k, op.ld_w, 128, 128);
  if (rc) return rc;
  rc = encode_8bit_2d(&tm_x, op.x, op.rows, op.k, op.ld_x, nt, 128);
  if (rc) return rc;
  static std::atomic<uint64_t> attr_done{0};
  auto kernel = gemm_i8_few_kernel<Epi>;
  rc = ensure_smem_attr(kernel, attr_done, kFewSmemBudget);
  if (rc) return rc;
  int sms = 0;
  rc = sm_count(&sms);
  if (rc) return rc;
  const int num_tiles = static_cast<int>((op.cols + 127) / 128);
  return launch_kernel(kernel, static_cast<unsigned>(num_tiles < 2 * sms ? num_tiles : 2 * sms), kFewThreads,
                       stages * stage_bytes + kOther, stream, op.quantised_here, tm_w, tm_x, ep, nt,
                       static_cast<int>((op.k + 127) / 128), stages, num_tiles, status);
}

template <typename OutT>
static int launch_product(const I8Operands& op, void* out, int64_t ld_out, int* status, cudaStream_t stream) {
  const I8Out p = {op.x_scale, op.w_scale, op.bias, op.bias_dtype, out, ld_out, static_cast<int>(op.rows),
                   static_cast<int>(op.cols)};
  if (op.rows <= kFewMaxTokens) return launch_few<FewStore<OutT>>(op, p, status, stream);
  return launch_gemm_i8<Int8StoreEpilogue<OutT>>(op.w, op.ld_w, op.x, op.ld_x, op.cols, op.rows, op.k, 16, p, status,
                                                 stream, op.quantised_here);
}

// Softmax partials of up to kFewMaxScored tokens, one per 128 columns.
static int launch_few_score(const I8Operands& op, const int64_t* target, float* partials, int64_t n_tiles, int* status,
                            cudaStream_t stream) {
  FewScore::Params ep = {};
  ep.op = {op.x_scale, op.w_scale, op.bias, op.bias_dtype, nullptr, 0, static_cast<int>(op.rows),
           static_cast<int>(op.cols)};
  ep.target = target;
  ep.partials = reinterpret_cast<float4*>(partials);
  ep.tile_stride = op.rows;
  ep.n_tiles = static_cast<int>(n_tiles);
  return launch_few<FewScore>(op, ep, status, stream);
}

template <bool kFull>
static int launch_score(const I8Operands& op, int64_t r0, int64_t n, const int64_t* target, float* partials,
                        int64_t tile_stride, int* status, cudaStream_t stream, bool overlap) {
  using Epi = Int8CEPartialsEpilogue<kFull>;
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
  // Few tokens go in one launch, whose partials cover 128 columns, whatever launch_rows is.
  const bool few = rows <= kFewMaxScored;
  const int64_t tile = few ? 128 : kBN;
  const int64_t n_tiles = vocab_size > 0 ? (vocab_size + tile - 1) / tile : 0;
  const int64_t step = few || launch_rows >= rows ? rows : launch_rows;
  FRX_CHECK_RANGE(target, rows * 8, "frx_i8_ce_entropy: target");
  FRX_CHECK_RANGE(ce, rows * 4, "frx_i8_ce_entropy: ce");
  FRX_CHECK_RANGE(entropy, rows * 4, "frx_i8_ce_entropy: entropy");
  FRX_CHECK_RANGE(lse, rows * 4, "frx_i8_ce_entropy: lse");
  FRX_CHECK_RANGE(log_probs, rows * 4, "frx_i8_ce_entropy: log_probs");
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
    rc = few ? launch_few_score(op, target, partials, n_tiles, status, st)
         : bias != nullptr || !op.quantised_here
             ? launch_score<true>(op, r0, n, target, partials, step, status, st, overlap)
             : launch_score<false>(op, r0, n, target, partials, step, status, st, overlap);
    if (rc) return rc;
    auto at = [r0](float* p) { return p == nullptr ? nullptr : p + r0; };
    rc = launch_finalize_dep(partials, n_tiles, n, step, target + r0, vocab_size, ignore_index, at(ce), at(entropy),
                             at(lse), at(log_probs), status, st);
    if (rc) return rc;
  }
  return FRX_OK;
}
