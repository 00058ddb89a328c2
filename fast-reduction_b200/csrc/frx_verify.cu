// Verification of drafted tokens against the target model's logits (speculative sampling: Leviathan,
// Kalman, Matias 2023; Chen et al. 2023), from given random numbers.
//
// Sequence b drafted tokens d_0 .. d_{n-1}; logits row i of the sequence is the target's distribution
// for the token at place i (n + 1 rows). With p_i = softmax(z_i / T_b) and draft probabilities q_i:
//   d_i is accepted while u_i q_i(d_i) < p_i(d_i)     (q_i(d_i) = 1 without draft probabilities)
//   a = number accepted; the next token is drawn from
//     w = max(p_a - q_a, 0)   after a rejection (without q: p_a with d_a taken out; p_a when nothing
//                             is left of w),
//     w = p_n                 when all were accepted,
//   as the first j with w_j > 0 and  sum_{k <= j} w_k > r sum_k w_k.
// T < 1e-6 (or NaN) is greedy: d_i is accepted while it equals argmax z_i (lowest index of a tie), and
// the next token is the argmax. NaN logits count as -inf, +inf as the largest float, negative or NaN
// draft probabilities as 0.
//
// Two launches:
//   stats   one warp per (row, 2048 columns): max, sum of exp((z - max) / T) and the index of the max.
//           Reads every logit once: HBM-bound.
//   sample  one cluster of 8 CTAs per sequence: merges the row statistics, decides a, then draws from
//           the chosen row. Running sums and probabilities are in 64 bits: which token's interval a
//           number falls in is a comparison over up to V borders, and sums in 32 bits would move each
//           border by 1e-7, enough to change a token about once in a hundred rows at V = 128256.
#include <cmath>

#include "frx_epilogue.cuh"
#include "frx_host.cuh"

namespace frx {

constexpr int kVfyChunk = 2048;  // columns per statistics partial
constexpr int kVfyThreads = 256;
constexpr int kVfyWarps = kVfyThreads / 32;
constexpr int kVfyCluster = 8;
constexpr float kVfyMinTemp = 1e-6f;
constexpr float kVfyMaxTemp = 1e6f;
constexpr float kFltMax = 3.402823466e38f;

// NaN counts as masked, +inf as the largest finite value (so that differences stay numbers).
__device__ __forceinline__ float clean_logit(float z) { return z == z ? fminf(z, kFltMax) : -INFINITY; }

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }

// Eight consecutive values as floats (16-byte aligned when vec).
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, int64_t n_valid, float fill, float (&v)[8]) {
  if (vec && n_valid >= 8) {
    if (sizeof(T) == 4) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(p));
      const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2(w[i], std::is_same<T, __half>::value);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n_valid ? to_f32<T>(p[i]) : fill;
  }
}

struct VerifyArgs {
  const void* logits;
  int64_t ld_logits;
  int logits_vec;
  const int64_t* drafts;
  const int64_t* cu;
  const float* uniforms;
  const float* final_uniforms;
  const void* q;  // [n_drafts, vocab] or null
  int64_t ld_q;
  int q_vec;
  const float* temperature;  // [batch] or null
  float temperature_all;
  int64_t batch;
  int64_t n_drafts;
  int64_t vocab;
  int n_chunks;
  float4* partials;  // [rows, n_chunks]: max, sum of exp, index of the max (int bits), unused
  int64_t* accepted;
  int64_t* tokens;
  float* log_probs;
  int* status;
};

struct SeqTemp {
  float t;      // the temperature the probabilities use (1 for greedy)
  bool greedy;
};

__device__ __forceinline__ SeqTemp seq_temp(const VerifyArgs& a, int64_t b) {
  const float t = a.temperature != nullptr ? __ldg(a.temperature + b) : a.temperature_all;
  SeqTemp s;
  s.greedy = !(t >= kVfyMinTemp);
  s.t = s.greedy ? 1.0f : fminf(t, kVfyMaxTemp);
  return s;
}

// Offsets as the kernels use them: clamped into the draft array whatever the caller passed.
__device__ __forceinline__ int64_t clamp_offset(int64_t x, int64_t n) { return x < 0 ? 0 : (x > n ? n : x); }

// Sequence that owns logits row `row`: the last b with cu[b] + b <= row.
__device__ __forceinline__ int64_t row_owner(const VerifyArgs& a, int64_t row) {
  int64_t lo = 0, hi = a.batch - 1;
  while (lo < hi) {
    const int64_t mid = (lo + hi + 1) >> 1;
    if (clamp_offset(__ldg(a.cu + mid), a.n_drafts) + mid <= row)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

template <typename T>
__global__ void __launch_bounds__(kVfyThreads) verify_stats_kernel(VerifyArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t rows = a.n_drafts + a.batch;
  const int64_t units = rows * a.n_chunks;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kVfyWarps + (threadIdx.x >> 5);
  if (unit >= units) return;
  const int64_t row = unit / a.n_chunks;
  const int chunk = static_cast<int>(unit - row * a.n_chunks);
  // rows behind the last sequence's are not read
  if (row >= clamp_offset(__ldg(a.cu + a.batch), a.n_drafts) + a.batch) return;
  const SeqTemp st = seq_temp(a, row_owner(a, row));
  const int64_t c0 = static_cast<int64_t>(chunk) * kVfyChunk;
  const int64_t n = min(static_cast<int64_t>(kVfyChunk), a.vocab - c0);
  const T* z = static_cast<const T*>(a.logits) + row * a.ld_logits + c0;
  constexpr int kIter = kVfyChunk / 256;
  float v[kIter][8];
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int64_t c = i * 256 + lane * 8;
    load8<T>(z + c, a.logits_vec != 0, n - c, -INFINITY, v[i]);
  }
#pragma unroll
  for (int i = 0; i < kIter; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[i][j] = clean_logit(v[i][j]);
      m = fmaxf(m, v[i][j]);
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float s = 0.0f;
  uint32_t idx = 0xFFFFFFFFu;
  if (m > -INFINITY) {
    const float k = kLog2e / st.t;
#pragma unroll
    for (int i = 0; i < kIter; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) s += ex2_approx((v[i][j] - m) * k);
    if (st.greedy) {
#pragma unroll
      for (int i = 0; i < kIter; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (v[i][j] == m) idx = min(idx, static_cast<uint32_t>(c0 + i * 256 + lane * 8 + j));
      idx = __reduce_min_sync(0xffffffffu, idx);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  }
  if (lane == 0) a.partials[row * a.n_chunks + chunk] = make_float4(m, s, __uint_as_float(idx), 0.0f);
}

// Statistics of one whole row, the same in every lane.
struct RowStats {
  float m;
  double s;
  uint32_t idx;
};

__device__ __forceinline__ RowStats merge_row(const VerifyArgs& a, int64_t row, float t, int lane) {
  const float4* p = a.partials + row * a.n_chunks;
  RowStats r{-INFINITY, 0.0, 0xFFFFFFFFu};
  for (int c = lane; c < a.n_chunks; c += 32) r.m = fmaxf(r.m, p[c].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) r.m = fmaxf(r.m, __shfl_xor_sync(0xffffffffu, r.m, o));
  if (r.m == -INFINITY) return r;
  for (int c = lane; c < a.n_chunks; c += 32) {
    const float4 v = p[c];
    if (v.x == -INFINITY) continue;
    r.s += static_cast<double>(v.y) * exp((static_cast<double>(v.x) - r.m) / t);
    if (v.x == r.m) r.idx = min(r.idx, __float_as_uint(v.z));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) r.s += __shfl_xor_sync(0xffffffffu, r.s, o);
  r.idx = __reduce_min_sync(0xffffffffu, r.idx);
  return r;
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// Reads a double from the same shared-memory variable of CTA `rank` of the cluster.
__device__ __forceinline__ double ld_cluster_f64(const double* local, uint32_t rank) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(map_to_cta(smem_u32(local), rank)) : "memory");
  return v;
}

// What the next token is drawn from.
enum DrawMode : int { kDrawP = 0, kDrawWithout = 1, kDrawResidual = 2 };

struct DrawRow {
  const void* z;
  const void* q;
  double m;
  double inv_t;
  double inv_s;
  int64_t without;  // kDrawWithout: the token taken out
  int mode;
};

// Weights of eight consecutive columns from c (those below `end`; others 0).
template <typename T, typename Q>
__device__ __forceinline__ void weights8(const VerifyArgs& a, const DrawRow& d, int64_t c, int64_t end,
                                         double (&w)[8]) {
  float z[8], q[8];
  load8<T>(static_cast<const T*>(d.z) + c, a.logits_vec != 0, end - c, -INFINITY, z);
  if (d.mode == kDrawResidual) load8<Q>(static_cast<const Q*>(d.q) + c, a.q_vec != 0, end - c, 0.0f, q);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float zc = clean_logit(z[j]);
    double p = zc == -INFINITY ? 0.0 : exp((static_cast<double>(zc) - d.m) * d.inv_t) * d.inv_s;
    if (d.mode == kDrawResidual) p = fmax(p - static_cast<double>(fmaxf(q[j], 0.0f)), 0.0);
    if (d.mode == kDrawWithout && c + j == d.without) p = 0.0;
    w[j] = p;
  }
}

template <typename T, typename Q>
__global__ void __cluster_dims__(kVfyCluster, 1, 1) __launch_bounds__(kVfyThreads) verify_sample_kernel(VerifyArgs a) {
  __shared__ int s_pass[kVfyThreads];
  __shared__ float s_logp[kVfyThreads];
  __shared__ double s_warp[kVfyWarps];
  __shared__ double s_total[2];  // read by the other CTAs of the cluster; one per exchange
  __shared__ RowStats s_row;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t rank = cluster_cta_rank();
  const int64_t b = blockIdx.x / kVfyCluster;
  const int64_t c_lo = __ldg(a.cu + b), c_hi = __ldg(a.cu + b + 1);
  const int64_t lo = clamp_offset(c_lo, a.n_drafts);
  const int64_t hi = max(lo, clamp_offset(c_hi, a.n_drafts));
  const int64_t n = hi - lo;
  const int64_t row0 = lo + b;
  const bool first_thread = rank == 0 && threadIdx.x == 0;
  if (first_thread && (c_lo != lo || c_hi != hi || (b == 0 && lo != 0)) && a.status != nullptr)
    atomicOr(a.status, kStatusBadOffsets);
  const SeqTemp st = seq_temp(a, b);
  const T* logits = static_cast<const T*>(a.logits);

  // ---- how many drafts pass: kVfyWarps at a time, every CTA of the cluster for itself
  int64_t acc = n;
  for (int64_t i0 = 0; i0 < n && acc == n; i0 += kVfyWarps) {
    const int64_t i = i0 + warp;
    if (i < n) {
      const RowStats r = merge_row(a, row0 + i, st.t, lane);
      const int64_t d = __ldg(a.drafts + lo + i);
      const bool valid = d >= 0 && d < a.vocab;
      int pass = 0;
      float logp = 0.0f;
      if (valid && r.m > -INFINITY) {
        const float z = clean_logit(to_f32<T>(logits[(row0 + i) * a.ld_logits + d]));
        const double x = (static_cast<double>(z) - r.m) / st.t;
        logp = static_cast<float>(x - log(r.s));
        if (st.greedy) {
          pass = static_cast<uint32_t>(d) == r.idx;
        } else {
          const double qd =
              a.q == nullptr ? 1.0 : fmaxf(to_f32<Q>(static_cast<const Q*>(a.q)[(lo + i) * a.ld_q + d]), 0.0f);
          pass = static_cast<double>(__ldg(a.uniforms + lo + i)) * qd < exp(x) / r.s;
        }
      }
      if (lane == 0) {
        s_pass[warp] = valid ? pass : -1;
        s_logp[warp] = logp;
      }
    }
    __syncthreads();
    int64_t stop = -1;
    for (int w = 0; w < kVfyWarps && i0 + w < n; ++w)
      if (s_pass[w] != 1) {
        stop = w;
        break;
      }
    if (stop >= 0) acc = i0 + stop;
    if (rank == 0 && threadIdx.x < kVfyWarps && i0 + threadIdx.x < acc) {
      a.tokens[row0 + i0 + threadIdx.x] = __ldg(a.drafts + lo + i0 + threadIdx.x);
      a.log_probs[row0 + i0 + threadIdx.x] = s_logp[threadIdx.x];
    }
    if (first_thread && stop >= 0 && s_pass[stop] < 0 && a.status != nullptr) atomicOr(a.status, kStatusBadTarget);
    __syncthreads();
  }
  const int64_t row = row0 + acc;
  if (warp == 0) {
    const RowStats r = merge_row(a, row, st.t, lane);
    if (lane == 0) s_row = r;
  }
  if (rank == 0) {
    const int64_t last = b == a.batch - 1 ? a.n_drafts + a.batch - 1 : row0 + n;
    for (int64_t i = row + 1 + threadIdx.x; i <= last; i += kVfyThreads) {
      a.tokens[i] = -1;
      a.log_probs[i] = 0.0f;
    }
    if (b == 0) {
      for (int64_t i = threadIdx.x; i < row0; i += kVfyThreads) {
        a.tokens[i] = -1;
        a.log_probs[i] = 0.0f;
      }
    }
    if (threadIdx.x == 0) a.accepted[b] = acc;
  }
  __syncthreads();
  const RowStats rs = s_row;
  // uniform over the cluster: no CTA of it reaches the exchanges below
  if (rs.m == -INFINITY || st.greedy) {
    if (first_thread) {
      a.tokens[row] = rs.m == -INFINITY ? -1 : static_cast<int64_t>(rs.idx);
      a.log_probs[row] = rs.m == -INFINITY ? -INFINITY : static_cast<float>(-log(rs.s));
    }
    return;
  }

  // ---- draw from row `row`
  DrawRow d;
  d.z = logits + row * a.ld_logits;
  d.q = a.q == nullptr ? nullptr : static_cast<const Q*>(a.q) + (lo + acc) * a.ld_q;
  d.m = rs.m;
  d.inv_t = 1.0 / st.t;
  d.inv_s = 1.0;
  d.without = -1;
  d.mode = kDrawP;
  // columns of this CTA, and of each of its warps, in order
  const int64_t per_warp = (((a.vocab + kVfyCluster * kVfyWarps - 1) / (kVfyCluster * kVfyWarps)) + 255) / 256 * 256;
  const int64_t w_lo = min(a.vocab, (static_cast<int64_t>(rank) * kVfyWarps + warp) * per_warp);
  const int64_t w_hi = min(a.vocab, w_lo + per_warp);
  int exchange = 0;
  double total = 0.0, before = 0.0, mine = 0.0;
  // This warp's sum of weights (mine), the sum of all columns before this CTA's (before) and of all
  // columns (total).
  auto sum_weights = [&]() {
    mine = 0.0;
    for (int64_t c = w_lo + lane * 8; c < w_hi; c += 256) {
      double w[8];
      weights8<T, Q>(a, d, c, w_hi, w);
      mine += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
    }
    mine = warp_sum(mine);
    __syncthreads();
    if (lane == 0) s_warp[warp] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
      double t = 0.0;
      for (int w = 0; w < kVfyWarps; ++w) t += s_warp[w];
      s_total[exchange] = t;
    }
    cluster_sync_all();
    total = before = 0.0;
    for (uint32_t k = 0; k < kVfyCluster; ++k) {
      const double t = ld_cluster_f64(&s_total[exchange], k);
      if (k < rank) before += t;
      total += t;
    }
    exchange ^= 1;
  };
  if (acc < n && a.q != nullptr) {
    sum_weights();  // the softmax denominator in 64 bits
    d.inv_s = 1.0 / total;
    d.mode = kDrawResidual;
    sum_weights();
    if (!(total > 0.0)) {
      d.mode = kDrawP;
      sum_weights();
    }
  } else {
    if (acc < n) {
      d.mode = kDrawWithout;
      d.without = __ldg(a.drafts + lo + acc);
    }
    sum_weights();
    if (!(total > 0.0)) {
      d.mode = kDrawP;
      sum_weights();
    }
  }
  // x = r * total falls to the last warp with any weight whose columns start at or before x (so exactly
  // one takes it, whatever rounding does at the ends); that warp walks its columns again.
  const float rf = __ldg(a.final_uniforms + b);
  const double x = (rf >= 0.0f ? fmin(static_cast<double>(rf), 1.0) : 0.0) * total;
  double after = before;  // where the next CTA's columns start
  bool later = false;     // a later CTA has weight
  for (uint32_t k = rank; k < kVfyCluster; ++k) {
    const double t = ld_cluster_f64(&s_total[exchange ^ 1], k);
    if (k == rank)
      after += t;
    else
      later = later || t > 0.0;
  }
  double start = before, next = later ? after : INFINITY;
  {
    double run = before;
    bool found = false;
    for (int w = 0; w < kVfyWarps; ++w) {
      const double at = fmin(run, after);
      if (w == warp) start = at;
      if (w > warp && !found && s_warp[w] > 0.0) {
        next = at;
        found = true;
      }
      run += s_warp[w];
    }
  }
  const bool takes = mine > 0.0 && start <= x && x < next;
  if (takes) {
    double run = start;
    int64_t token = -1, last_live = -1;
    double zx = 0.0;
    for (int64_t c0 = w_lo; c0 < w_hi && token < 0; c0 += 256) {
      const int64_t c = c0 + lane * 8;
      double w[8];
      if (c < w_hi) {
        weights8<T, Q>(a, d, c, w_hi, w);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = 0.0;
      }
      double sum = 0.0;
      int live = -1;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sum += w[j];
        if (w[j] > 0.0) live = j;
      }
      double incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
      }
      double cur = run + (incl - sum);
      int hit = -1;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        cur += w[j];
        if (hit < 0 && w[j] > 0.0 && cur > x) hit = j;
      }
      const uint32_t hits = __ballot_sync(0xffffffffu, hit >= 0);
      const uint32_t lives = __ballot_sync(0xffffffffu, live >= 0);
      if (hits != 0) {
        const int l = __ffs(hits) - 1;
        token = c0 + l * 8 + __shfl_sync(0xffffffffu, hit, l);
      } else if (lives != 0) {
        const int l = 31 - __clz(lives);
        last_live = c0 + l * 8 + __shfl_sync(0xffffffffu, live, l);
      }
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (token < 0) token = last_live;
    if (lane == 0) {
      zx = (static_cast<double>(clean_logit(to_f32<T>(static_cast<const T*>(d.z)[token]))) - d.m) * d.inv_t;
      a.tokens[row] = token;
      a.log_probs[row] = static_cast<float>(zx - log(rs.s));
    }
  }
  cluster_sync_all();  // no CTA leaves while another may still read its sums
}

template <typename T, typename Q>
static int launch_verify(const VerifyArgs& a, cudaStream_t stream) {
  const int64_t rows = a.n_drafts + a.batch;
  const int64_t blocks = (rows * a.n_chunks + kVfyWarps - 1) / kVfyWarps;
  FRX_REQUIRE(blocks < (1ll << 31) && a.batch * kVfyCluster < (1ll << 31), FRX_ERR_INVALID_ARG,
              "frx_verify_drafts: problem too large (%lld rows, %lld columns)", (long long)rows, (long long)a.vocab);
  verify_stats_kernel<T><<<static_cast<unsigned>(blocks), kVfyThreads, 0, stream>>>(a);
  FRX_CUDA_CHECK(cudaGetLastError());
  verify_sample_kernel<T, Q><<<static_cast<unsigned>(a.batch * kVfyCluster), kVfyThreads, 0, stream>>>(a);
  FRX_CUDA_CHECK(cudaGetLastError());
  return FRX_OK;
}

template <typename T>
static int launch_verify_q(const VerifyArgs& a, int q_dtype, cudaStream_t stream) {
  if (q_dtype == FRX_DTYPE_BF16) return launch_verify<T, __nv_bfloat16>(a, stream);
  if (q_dtype == FRX_DTYPE_F16) return launch_verify<T, __half>(a, stream);
  return launch_verify<T, float>(a, stream);
}

}  // namespace frx

extern "C" int frx_verify_drafts(const void* logits, int dtype, int64_t ld_logits, const int64_t* drafts,
                                 const int64_t* cu_drafts, const float* uniforms, const float* final_uniforms,
                                 const void* draft_probs, int draft_probs_dtype, int64_t ld_draft_probs,
                                 const float* temperature, float temperature_all, int64_t batch, int64_t n_drafts,
                                 int64_t vocab, float* workspace, int64_t workspace_floats, int64_t* accepted,
                                 int64_t* tokens, float* log_probs, int* status, void* stream) {
  using namespace frx;
  FRX_REQUIRE(batch >= 0 && n_drafts >= 0 && vocab >= 1 && vocab < (1ll << 31) && batch < (1ll << 31) &&
                  n_drafts < (1ll << 31) && ld_logits >= vocab,
              FRX_ERR_INVALID_ARG, "frx_verify_drafts: bad sizes batch=%lld n_drafts=%lld vocab=%lld ld_logits=%lld",
              (long long)batch, (long long)n_drafts, (long long)vocab, (long long)ld_logits);
  FRX_REQUIRE(dtype == FRX_DTYPE_BF16 || dtype == FRX_DTYPE_F16 || dtype == FRX_DTYPE_F32, FRX_ERR_INVALID_ARG,
              "frx_verify_drafts: unknown logits dtype %d", dtype);
  FRX_REQUIRE(draft_probs == nullptr || ((draft_probs_dtype == FRX_DTYPE_BF16 || draft_probs_dtype == FRX_DTYPE_F16 ||
                                          draft_probs_dtype == FRX_DTYPE_F32) &&
                                         ld_draft_probs >= vocab),
              FRX_ERR_INVALID_ARG, "frx_verify_drafts: draft_probs need a dtype of BF16, F16 or F32 (got %d) and "
              "ld_draft_probs %lld >= vocab", draft_probs_dtype, (long long)ld_draft_probs);
  if (batch == 0) {
    FRX_REQUIRE(n_drafts == 0, FRX_ERR_INVALID_ARG, "frx_verify_drafts: %lld drafts of no sequence",
                (long long)n_drafts);
    return FRX_OK;
  }
  FRX_REQUIRE(logits != nullptr && cu_drafts != nullptr && final_uniforms != nullptr && workspace != nullptr &&
                  accepted != nullptr && tokens != nullptr && log_probs != nullptr &&
                  (n_drafts == 0 || (drafts != nullptr && uniforms != nullptr)),
              FRX_ERR_INVALID_ARG, "frx_verify_drafts: null pointer");
  const int64_t rows = n_drafts + batch;
  const int64_t n_chunks = (vocab + kVfyChunk - 1) / kVfyChunk;
  FRX_REQUIRE(aligned16(workspace) && workspace_floats >= 4 * rows * n_chunks, FRX_ERR_INVALID_ARG,
              "frx_verify_drafts: workspace must be 16-byte aligned with 4 * %lld * %lld floats (got %lld)",
              (long long)rows, (long long)n_chunks, (long long)workspace_floats);
  const int64_t esz = dtype == FRX_DTYPE_F32 ? 4 : 2;
  const int64_t qsz = draft_probs_dtype == FRX_DTYPE_F32 ? 4 : 2;
  FRX_CHECK_RANGE(logits, matrix_bytes(rows, vocab, ld_logits, esz), "frx_verify_drafts: logits");
  FRX_CHECK_RANGE(draft_probs, matrix_bytes(n_drafts, vocab, ld_draft_probs, qsz), "frx_verify_drafts: draft_probs");
  FRX_CHECK_RANGE(drafts, n_drafts * 8, "frx_verify_drafts: drafts");
  FRX_CHECK_RANGE(cu_drafts, (batch + 1) * 8, "frx_verify_drafts: cu_drafts");
  FRX_CHECK_RANGE(uniforms, n_drafts * 4, "frx_verify_drafts: uniforms");
  FRX_CHECK_RANGE(final_uniforms, batch * 4, "frx_verify_drafts: final_uniforms");
  FRX_CHECK_RANGE(temperature, batch * 4, "frx_verify_drafts: temperature");
  FRX_CHECK_RANGE(workspace, 16 * rows * n_chunks, "frx_verify_drafts: workspace");
  FRX_CHECK_RANGE(accepted, batch * 8, "frx_verify_drafts: accepted");
  FRX_CHECK_RANGE(tokens, rows * 8, "frx_verify_drafts: tokens");
  FRX_CHECK_RANGE(log_probs, rows * 4, "frx_verify_drafts: log_probs");
  VerifyArgs a = {};
  a.logits = logits;
  a.ld_logits = ld_logits;
  a.logits_vec = aligned16(logits) && (ld_logits * esz) % 16 == 0;
  a.drafts = drafts;
  a.cu = cu_drafts;
  a.uniforms = uniforms;
  a.final_uniforms = final_uniforms;
  a.q = draft_probs;
  a.ld_q = ld_draft_probs;
  a.q_vec = aligned16(draft_probs) && (ld_draft_probs * qsz) % 16 == 0;
  a.temperature = temperature;
  a.temperature_all = temperature_all;
  a.batch = batch;
  a.n_drafts = n_drafts;
  a.vocab = vocab;
  a.n_chunks = static_cast<int>(n_chunks);
  a.partials = reinterpret_cast<float4*>(workspace);
  a.accepted = accepted;
  a.tokens = tokens;
  a.log_probs = log_probs;
  a.status = status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == FRX_DTYPE_BF16) return launch_verify_q<__nv_bfloat16>(a, draft_probs_dtype, st);
  if (dtype == FRX_DTYPE_F16) return launch_verify_q<__half>(a, draft_probs_dtype, st);
  return launch_verify_q<float>(a, draft_probs_dtype, st);
}
