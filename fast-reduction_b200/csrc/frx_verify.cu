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
// the next token is the argmax. NaN logits count as -inf, +inf as the largest finite one, negative or NaN
// draft probabilities as 0.
//
// Two launches:
//   stats   one warp per (row, 2048 or more columns): max, sum of exp((z - max) / T) and the index of the max.
//           Reads every logit once. V = 128256 bf16: 288 rows 19 us (3.9 TB/s), 1150 rows 57 us (5.2 TB/s); exponentials
//           and loads take turns (a ring of asynchronous copies and smaller or more blocks were no faster).
//   sample  one cluster of 1 to 8 CTAs per sequence: merges the row statistics, decides a, then draws from
//           the chosen row. Running sums and probabilities are in 64 bits: which token's interval a
//           number falls in is a comparison over up to V borders, and sums in 32 bits would move each
//           border by 1e-7, enough to change a token about once in a hundred rows at V = 128256. Acceptance is one
//           comparison, which the statistics' fp32 sum decides unless the two sides are closer than that sum's
//           error bound (stats_sum_error, 7e-5; one draft in some ten thousand): then the row is summed in 64 bits.
//           It is bound by latency: a cluster waits for its first CTA's decision (the largest stall is the barrier,
//           issue slots and the 64-bit pipe are below 30 % on average), and its passes are long chains of
//           64-bit operations, so the exponential is a short one of its own (exp2_scaled below). 64 sequences of
//           V = 128256 with draft probabilities: 56 us in all; per cluster 5 us for the decision, 7 for a pass over a
//           row, 3 for the search.
#include <cmath>
#include <cstring>
#include <type_traits>

#include "frx_epilogue.cuh"
#include "frx_host.cuh"

namespace frx {

constexpr int kVfyChunk = FRX_VERIFY_CHUNK;  // least columns per statistics partial (up to 7 of a first one lie before the row)
constexpr int kVfyThreads = 256;
constexpr int kVfyWarps = kVfyThreads / 32;
constexpr int kVfyMaxCluster = 8;
constexpr int kVfyMaxGroups = 16;  // groups of columns per warp whose lane sums are kept for the search
constexpr float kVfyMinTemp = 1e-6f;
constexpr float kVfyMaxTemp = 1e6f;
constexpr float kFltMax = 3.402823466e38f;

// NaN counts as masked (fmaxf drops it), +inf as a finite value no other logit exceeds (so that differences stay
// numbers): the largest float, or for 16-bit logits the largest bf16 value, whose low 16 bits are zero.
template <typename T>
__device__ __forceinline__ float clean_logit(float z) {
  return fminf(fmaxf(z, -INFINITY), sizeof(T) == 4 ? kFltMax : 3.38953139e38f);
}

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }

// 2^(j / 1024) = coarse[j / 32] * fine[j % 32], rounded to 64 bits each.
struct Exp2Table {
  double coarse[32], fine[32];
};
static Exp2Table make_exp2_table() {
  Exp2Table t;
  for (int j = 0; j < 32; ++j) {
    t.coarse[j] = static_cast<double>(exp2l(static_cast<long double>(j) / 32.0L));
    t.fine[j] = static_cast<double>(exp2l(static_cast<long double>(j) / 1024.0L));
  }
  return t;
}
constexpr int kExp2Entries = 1024;

// scale * 2^(a b / 1024) for -1024 * 1000 <= a b < 1024, table[j] = scale * 2^(j / 1024): by table and polynomial
// (P. T. P. Tang, "Table-driven implementation of the exponential function in IEEE floating-point
// arithmetic", 1989). a b = 1024 n + j + f with |f| <= 1/2; 2^(f / 1024) = e^x with |x| <= h = ln 2 / 2048 as
// 1 + (1 + h^2 / 8) x + x^2 / 2, the Taylor terms with the cubic one economised (Lanczos: x^3 is (3/4) h^2 x to
// within h^3 / 4 there), which is 1.6e-12 off at most and odd in x, so that sums over many values gain more.
// Adding 1.5 * 2^52 rounds to an integer. Seven 64-bit operations; a table of 64 entries took four more.
// Outside the range the result is some number, which the caller drops.
__device__ __forceinline__ double exp2_scaled(double a, double b, const double* table) {
  constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52
  constexpr double kLn = 0.6931471805599453094 / kExp2Entries;
  constexpr double c1 = kLn * (1.0 + kLn * kLn / 32), c2 = kLn * kLn / 2;  // h = kLn / 2
  const double r = fma(a, b, kMagic);
  const int k = __double2loint(r);
  const double f = fma(a, b, kMagic - r);
  const double g = f * fma(f, c2, c1);
  const double t = table[k & (kExp2Entries - 1)];
  // times 2^(k >> 10) through the exponent field
  const double s = __hiloint2double((k & ~(kExp2Entries - 1)) * (1 << 10) + __double2hiint(t), __double2loint(t));
  return fma(s, g, s);
}

// An fp32 value in 64 bits by its bits (conversions run at a quarter of the 64-bit pipe's rate). Zero and
// subnormals come out as up to 2^-126 instead, which no logit notices. T: the type the value was read as (the
// low word is zero for the 16-bit ones).
template <typename T>
__device__ __forceinline__ double widen(float x) {
  const int b = __float_as_int(x);
  return __hiloint2double(((b >> 3) & 0x8fffffff) + (896 << 20), sizeof(T) == 4 ? b << 29 : 0);
}

// The same for a draft probability, with negative values, NaN and subnormals as 0 (infinity: above every
// probability).
template <typename T>
__device__ __forceinline__ double widen_prob(float x) {
  const int b = __float_as_int(fmaxf(x, 0.0f));
  return __hiloint2double(b >= 0x800000 ? (b >> 3) + (896 << 20) : 0, sizeof(T) == 4 ? b << 29 : 0);
}

// Eight values of a row as they lie in memory (two per word for 16-bit types).
template <typename T>
struct Vec8 {
  static constexpr int kWords = sizeof(T) == 4 ? 8 : 4;
  uint32_t w[kWords];

  __device__ __forceinline__ void load(const T* p) {  // 16-byte aligned
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    if (sizeof(T) == 4) {
      const uint4 b = __ldg(reinterpret_cast<const uint4*>(p) + 1);
      w[kWords - 4] = b.x; w[kWords - 3] = b.y; w[kWords - 2] = b.z; w[kWords - 1] = b.w;
    }
  }
  // Values p[j * step] for the j with lo <= j * step < hi; `fill` (bits of a T) for the others.
  __device__ __forceinline__ void load_some(const T* p, int step, int lo, int hi, uint32_t fill) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t x = fill;
      if (j * step >= lo && j * step < hi)
        x = sizeof(T) == 4 ? __ldg(reinterpret_cast<const uint32_t*>(p) + j * step)
                           : __ldg(reinterpret_cast<const uint16_t*>(p) + j * step);
      if (sizeof(T) == 4)
        w[j % kWords] = x;
      else
        w[j / 2] = (j & 1) ? (w[j / 2] | (x << 16)) : x;
    }
  }
  __device__ __forceinline__ float at(int j) const {
    if (sizeof(T) == 4) return __uint_as_float(w[j % kWords]);
    const float2 f = unpack2(w[j / 2], std::is_same<T, __half>::value);
    return (j & 1) ? f.y : f.x;
  }
  // The largest value; NaN is dropped (all NaN: NaN).
  __device__ __forceinline__ float max() const {
    if (sizeof(T) == 4)
      return fmaxf(fmaxf(fmaxf(at(0), at(1)), fmaxf(at(2), at(3))), fmaxf(fmaxf(at(4), at(5)), fmaxf(at(6), at(7))));
    uint32_t m;
    if (std::is_same<T, __half>::value) {
      __half2 h[4];
      memcpy(h, w, sizeof(h));
      const __half2 x = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
      memcpy(&m, &x, sizeof(m));
    } else {
      __nv_bfloat162 h[4];
      memcpy(h, w, sizeof(h));
      const __nv_bfloat162 x = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
      memcpy(&m, &x, sizeof(m));
    }
    const float2 f = unpack2(m, std::is_same<T, __half>::value);
    return fmaxf(f.x, f.y);
  }
  __device__ __forceinline__ void mask(int j) {  // value j becomes -inf
    if (sizeof(T) == 4)
      w[j % kWords] = kNegInf;
    else
      w[j / 2] = (j & 1) ? ((w[j / 2] & 0xffffu) | (kNegInf << 16)) : ((w[j / 2] & 0xffff0000u) | kNegInf);
  }
  static constexpr uint32_t kNegInf =
      sizeof(T) == 4 ? 0xff800000u : (std::is_same<T, __half>::value ? 0xfc00u : 0xff80u);
};

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
  int chunk_cols;  // columns per statistics partial: kVfyChunk times a power of two
  int row_step;    // stats: rows of a sequence are dealt to this many blocks
  int early;       // stats: the sample kernel may start beside this one
  int strip_step;  // sample: 256-column strips per group of columns
  double sum_error;  // relative error of a row's sum of the statistics
  Exp2Table exp2;
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

// The running maximum (from -FLT_MAX), sum of exp((z - m) / T) and index of the maximum of one lane or row; s = 0
// says that nothing but masked logits was seen.
struct RowStats {
  float m;
  float s;
  uint32_t idx;
};

__device__ __forceinline__ void join_stats(RowStats& r, const RowStats& o, float k) {
  const float m = fmaxf(r.m, o.m);
  // the lowest index of a tie; a side without a live logit has none
  if (o.s > 0.0f && (r.s == 0.0f || o.m > r.m || (o.m == r.m && o.idx < r.idx))) r.idx = o.idx;
  r.s = r.s * ex2_approx((r.m - m) * k) + o.s * ex2_approx((o.m - m) * k);
  r.m = m;
}

// Adds 8 N values to a lane's statistics: those of N vectors 256 columns apart, the first one's column is col.
template <typename T, int N>
__device__ __forceinline__ void add_vectors(RowStats& r, const Vec8<T> (&raw)[N], float k, bool greedy, uint32_t col) {
  float v[8 * N], top = raw[0].max();
#pragma unroll
  for (int i = 1; i < N; ++i) top = fmaxf(top, raw[i].max());
#pragma unroll
  for (int j = 0; j < 8 * N; ++j) v[j] = raw[j / 8].at(j % 8);
  float sum;
  auto add = [&]() {
    const float m = fmaxf(r.m, top), was = r.s * ex2_approx((r.m - m) * k);
    const uint64_t neg = pack_f32x2(-m, -m), k2 = pack_f32x2(k, k);
    uint64_t s2 = 0, s3 = 0;
#pragma unroll
    for (int j = 0; j < 8 * N; j += 2) {
      float a0, a1;
      unpack_f32x2(mul_f32x2(add_f32x2(pack_f32x2(v[j], v[j + 1]), neg), k2), a0, a1);
      const uint64_t e = pack_f32x2(ex2_approx(a0), ex2_approx(a1));
      if (j & 2)
        s3 = add_f32x2(s3, e);
      else
        s2 = add_f32x2(s2, e);
    }
    float f0, f1;
    unpack_f32x2(add_f32x2(s2, s3), f0, f1);
    sum = f0 + f1;
    if (sum <= 8.5f * N) {
      if (greedy && (top > r.m || (r.s == 0.0f && top == r.m))) {
#pragma unroll
        for (int j = 8 * N - 1; j >= 0; --j)
          if (v[j] == top) r.idx = col + (j / 8) * 256 + j % 8;
      }
      r.s = was + sum;
      r.m = m;
    }
  };
  // No test of the single values: each adds at most 1, so a NaN or +inf among them shows in the sum, and they are
  // cleaned then.
  add();
  if (!(sum <= 8.5f * N)) {
#pragma unroll
    for (int j = 0; j < 8 * N; ++j) v[j] = clean_logit<T>(v[j]);
    top = clean_logit<T>(top);
    add();
  }
}

// grid: (chunks / warps per CTA, sequences, row_step). A warp takes one chunk of every row_step-th row of its
// sequence, so that its offsets and temperature are one round of loads, whatever the sequences' lengths. A
// chunk starts on a 16-byte boundary: chunk c of a row whose first value lies `head` values past one covers the
// columns [n c - head, n (c + 1) - head), n = chunk_cols. 512 or 1024 columns at a time, the next ones requested under the
// current ones'; each lane keeps a maximum and a sum of its own, joined by shuffles at the end.
template <typename T>
__global__ void __launch_bounds__(kVfyThreads) verify_stats_kernel(const __grid_constant__ VerifyArgs a) {
  if (a.early) grid_dep_launch();
  const int lane = threadIdx.x & 31;
  const int chunk = static_cast<int>(blockIdx.x) * kVfyWarps + static_cast<int>(threadIdx.x >> 5);
  if (chunk >= a.n_chunks) return;
  for (int64_t b = blockIdx.y; b < a.batch; b += gridDim.y) {
    const int64_t lo = clamp_offset(__ldg(a.cu + b), a.n_drafts);
    const int64_t hi = max(lo, clamp_offset(__ldg(a.cu + b + 1), a.n_drafts));
    const SeqTemp st = seq_temp(a, b);
    const float k = kLog2e / st.t;
    for (int64_t row = lo + b + blockIdx.z; row <= hi + b; row += a.row_step) {
      const T* z = static_cast<const T*>(a.logits) + row * a.ld_logits;
      const int head = static_cast<int>((reinterpret_cast<uintptr_t>(z) & 15u) / sizeof(T));
      const int64_t first = static_cast<int64_t>(chunk) * a.chunk_cols - head;  // column of the chunk's first vector
      const int64_t end = min(a.vocab, first + a.chunk_cols);
      RowStats r{-kFltMax, 0.0f, 0xFFFFFFFFu};
      int c = static_cast<int>(first) + lane * 8;
      const T* zp = z + c;
      const int vocab = static_cast<int>(a.vocab);
      auto load = [&](int ahead, Vec8<T>& v) {
        const int at = c + ahead;
        if (at >= 0 && at + 8 <= vocab)
          v.load(zp + ahead);
        else
          v.load_some(zp + ahead, 1, -at, vocab - at, Vec8<T>::kNegInf);
      };
      constexpr int kVec = sizeof(T) == 4 ? 2 : 4;  // 64 bytes in flight per lane
      Vec8<T> nxt[kVec];
#pragma unroll
      for (int i = 0; i < kVec; ++i) load(256 * i, nxt[i]);
#pragma unroll 1
      for (int n = static_cast<int>(end - first); n > 0; n -= 256 * kVec) {
        Vec8<T> cur[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) cur[i] = nxt[i];
        if (n > 256 * kVec) {
#pragma unroll
          for (int i = 0; i < kVec; ++i) load(256 * (kVec + i), nxt[i]);
        }
        add_vectors<T, kVec>(r, cur, k, st.greedy, static_cast<uint32_t>(c));
        c += 256 * kVec;
        zp += 256 * kVec;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        RowStats x;
        x.m = __shfl_xor_sync(0xffffffffu, r.m, o);
        x.s = __shfl_xor_sync(0xffffffffu, r.s, o);
        x.idx = __shfl_xor_sync(0xffffffffu, r.idx, o);
        join_stats(r, x, k);
      }
      if (lane == 0) a.partials[row * a.n_chunks + chunk] = make_float4(r.m, r.s, __uint_as_float(r.idx), 0.0f);
    }
  }
  if (!a.early) grid_dep_launch();
}

// Statistics of one whole row, the same in every lane.
__device__ __forceinline__ RowStats merge_row(const VerifyArgs& a, int64_t row, float t, int lane) {
  const float4* p = a.partials + row * a.n_chunks;
  const float k = kLog2e / t;
  RowStats r{-kFltMax, 0.0f, 0xFFFFFFFFu};
#pragma unroll 1
  for (int c0 = lane; c0 < a.n_chunks; c0 += 128) {
    float4 v[4];  // four loads in flight
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = c0 + 32 * i < a.n_chunks ? ld_dep_v4(p + c0 + 32 * i) : make_float4(-kFltMax, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) join_stats(r, RowStats{v[i].x, v[i].y, __float_as_uint(v[i].z)}, k);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    RowStats x;
    x.m = __shfl_xor_sync(0xffffffffu, r.m, o);
    x.s = __shfl_xor_sync(0xffffffffu, r.s, o);
    x.idx = __shfl_xor_sync(0xffffffffu, r.idx, o);
    join_stats(r, x, k);
  }
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

// How many drafts of a sequence passed, and the maximum and sum of the row that its next token comes from.
struct __align__(16) Decision {
  int64_t acc;
  float m, s;
};

// The same variable of CTA `rank` of the cluster.
__device__ __forceinline__ Decision ld_cluster_decision(const Decision* local, uint32_t rank) {
  Decision d;
  asm volatile("{\n\t.reg .b64 t;\n\tld.shared::cluster.v2.b64 {%0, t}, [%3];\n\tmov.b64 {%1, %2}, t;\n\t}"
               : "=l"(d.acc), "=f"(d.m), "=f"(d.s)
               : "r"(map_to_cta(smem_u32(local), rank))
               : "memory");
  return d;
}

constexpr int kPassOpen = 2;  // a draft whose acceptance the fp32 sum of its row cannot decide

// What the next token is drawn from.
enum DrawMode : int { kDrawP = 0, kDrawWithout = 1, kDrawResidual = 2 };

struct DrawRow {
  const void* z;
  const void* q;
  double m;
  double scale;  // 1024 log2(e) / T: exp((z - m) / T) = 2^((z - m) scale / 1024)
  float floor;   // logits below have weight 0: the least float from m - 680 T on, where exp is 4e-296
  int without;  // kDrawWithout: the token taken out, else -1
  int mode;
};

// Weight of one column of the drawn row from its logit and (kResidual) draft probability. `live` false: the
// column has no weight and the value returned is some number. A residual of exactly 0 counts as live.
template <typename T, typename Q, bool kResidual>
__device__ __forceinline__ double draw_weight(const DrawRow& d, const double* table, float z, float q, bool& live) {
  constexpr float kCap = sizeof(T) == 4 ? kFltMax : 3.38953139e38f;  // as clean_logit
  double w = exp2_scaled(widen<T>(fminf(z, kCap)) - d.m, d.scale, table);
  live = z >= d.floor;  // false for NaN
  if (kResidual) {
    w -= widen_prob<Q>(q);
    live = live && __double2hiint(w) >= 0;
  }
  return w;
}

// Eight columns of the drawn row as they are read: `n` of them from zp and qp on with that step are there (others
// count as masked). vec: whole vectors may be loaded (step 1).
template <typename T, typename Q, bool kResidual>
struct DrawCols {
  Vec8<T> z;
  Vec8<Q> q;
  __device__ __forceinline__ void load(const T* zp, const Q* qp, int step, int n, bool vec) {
    if (vec && n >= 8) {
      z.load(zp);
      if (kResidual) q.load(qp);
    } else {
      z.load_some(zp, step, 0, n, Vec8<T>::kNegInf);
      if (kResidual) q.load_some(qp, step, 0, n, 0);
    }
  }
};

// kDrawWithout: masks the token that is taken out in the columns c + j * step, if it is among them.
template <typename T>
__device__ __forceinline__ void mask_without(const DrawRow& d, Vec8<T>& z, int c, int step) {
  if (d.without >= c && d.without < c + 8 * step) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j * step == d.without) z.mask(j);
  }
}

// Sum of this lane's weights over the columns [lo, hi) of its warp; the sums over each group of group_cols columns
// go to s_lane[group][thread].
template <typename T, typename Q, bool kResidual>
__device__ __forceinline__ double sum_columns(const VerifyArgs& a, const DrawRow& d, const double* table, int lo, int hi,
                                              int group_cols, double (*s_lane)[kVfyThreads]) {
  const int lane = threadIdx.x & 31;
  const bool vec = a.logits_vec != 0 && (!kResidual || a.q_vec != 0);
  // whole vectors, or coalesced single values (a sum does not care for the order)
  const int step = vec ? 1 : 32;
  int c = lo + (vec ? lane * 8 : lane);
  const T* zp = static_cast<const T*>(d.z) + c;
  const Q* qp = static_cast<const Q*>(d.q) + c;
  DrawCols<T, Q, kResidual> nxt;
  nxt.load(zp, qp, step, hi - c, vec);
  double all = 0.0;
  int g = 0;
#pragma unroll 1
  for (int g0 = lo; g0 < hi; g0 += group_cols, ++g) {
    const int strips = (min(hi - g0, group_cols) + 255) >> 8;
    double sum = 0.0, sum1 = 0.0;
#pragma unroll 1
    for (int i = 0; i < strips; ++i) {
      DrawCols<T, Q, kResidual> cur = nxt;
      zp += 256;
      qp += 256;
      nxt.load(zp, qp, step, hi - c - 256, vec);  // behind the last column nothing is read
      if (!kResidual) mask_without(d, cur.z, c, step);
      c += 256;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        bool live;
        const double w = draw_weight<T, Q, kResidual>(d, table, cur.z.at(j), kResidual ? cur.q.at(j) : 0.0f, live);
        if (live) {
          if (j & 1)
            sum1 += w;
          else
            sum += w;
        }
      }
    }
    sum += sum1;
    s_lane[g][threadIdx.x] = sum;
    all += sum;
  }
  return all;
}

// The part of a row's fp32 sum s of exp((z - m) / T) by which that sum may be off, with h = 2^-24: exponents
// a = (z - m) k, each of 4 roundings, where |a| <= 55 (what lies below adds less than 2^30 2^-55): 4 * 55 ln 2 = 153 h; the
// same again for the rises of the maximum, 4 h for ex2.approx, 10 h for a lane's sum of one load, 6 h for each of up to 64
// loads and 6 h for each of 14 + n_chunks / 32 joins: below (800 + n_chunks) h.
inline double stats_sum_error(int n_chunks) { return (1024.0 + n_chunks) / (1 << 24); }

// Row `z` for draws and sums over all its tokens; m: its maximum.
__device__ __forceinline__ DrawRow draw_row(const void* z, float m, float t) {
  DrawRow d;
  d.z = z;
  d.q = nullptr;
  d.m = m;
  // rounded up: at 1500 and T = 1e-6 a step of fp32 is 122 T, and a cutoff rounded down would let in logits below the
  // range of exp2_scaled, whose results are some number there
  d.floor = __fmaf_ru(-680.0f, t, m);
  d.scale = kExp2Entries * 1.4426950408889634074 / t;
  d.without = -1;
  d.mode = kDrawP;
  return d;
}

// Sum of exp((z - m) / T) over a whole row in 64 bits, by all threads of the CTA (table: of scale 1). Out of line: one draft
// in some ten thousand needs it.
template <typename T>
__device__ __noinline__ double row_sum_f64(const VerifyArgs& a, const void* z, float m, float t, const double* table,
                                           double (*s_lane)[kVfyThreads], double* s_warp) {
  const DrawRow d = draw_row(z, m, t);
  constexpr int kSpan = 256 * kVfyWarps;
  const int strips = static_cast<int>((a.vocab + kSpan - 1) / kSpan);
  const int group_cols = 256 * ((strips + kVfyMaxGroups - 1) / kVfyMaxGroups);
  const int64_t per_warp = ((a.vocab + kVfyWarps - 1) / kVfyWarps + group_cols - 1) / group_cols * group_cols;
  const int warp = threadIdx.x >> 5;
  const int lo = static_cast<int>(min(a.vocab, warp * per_warp));
  const int hi = static_cast<int>(min(a.vocab, lo + per_warp));
  const double mine = warp_sum(sum_columns<T, float, false>(a, d, table, lo, hi, group_cols, s_lane));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s_warp[warp] = mine;
  __syncthreads();
  double total = 0.0;
  for (int w = 0; w < kVfyWarps; ++w) total += s_warp[w];
  return total;
}

template <typename T, typename Q>
__global__ void __launch_bounds__(kVfyThreads, 3) verify_sample_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ int s_pass[kVfyWarps];
  __shared__ double s_x[kVfyWarps];
  __shared__ double s_uq[kVfyWarps];
  __shared__ Decision s_decision;
  __shared__ double s_warp[kVfyWarps];
  __shared__ double s_total[2];  // read by the other CTAs of the cluster; one per exchange
  __shared__ RowStats s_rows[kVfyWarps];
  __shared__ double s_exp2[kExp2Entries];  // over the softmax denominator where weights are probabilities
  __shared__ double s_lane[kVfyMaxGroups][kVfyThreads];  // a lane's sum over each of its warp's groups of columns
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t rank = cluster_cta_rank(), ctas = cluster_cta_count();
  const int64_t b = blockIdx.x / ctas;
  for (int j = threadIdx.x; j < kExp2Entries; j += kVfyThreads) s_exp2[j] = a.exp2.coarse[j >> 5] * a.exp2.fine[j & 31];
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

  // ---- how many drafts pass: the cluster's first CTA decides, kVfyWarps rows at a time, and hands the result to
  // the others through its shared memory. What does not depend on the statistics is loaded before the wait for
  // them. Row n has no draft to pass.
  if (rank == 0) {
    int64_t acc = -1;
#pragma unroll 1
    for (int64_t i0 = 0; acc < 0; i0 += kVfyWarps) {
      const int64_t i = i0 + warp;
      if (i <= n) {
        int64_t d = -1;
        bool valid = false;
        float z = -INFINITY, qd = 1.0f, u = 0.0f;
        if (i < n) {
          d = __ldg(a.drafts + lo + i);
          u = __ldg(a.uniforms + lo + i);
          valid = d >= 0 && d < a.vocab;
          if (valid) {
            z = clean_logit<T>(to_f32<T>(logits[(row0 + i) * a.ld_logits + d]));
            if (a.q != nullptr) qd = fmaxf(to_f32<Q>(static_cast<const Q*>(a.q)[(lo + i) * a.ld_q + d]), 0.0f);
          }
        }
        grid_dep_wait();
        const RowStats r = merge_row(a, row0 + i, st.t, lane);
        if (lane == 0) {
          const double x = (static_cast<double>(z) - r.m) / st.t;
          int pass = 0;
          if (valid && r.s > 0.0f) {
            if (st.greedy) {
              pass = static_cast<uint32_t>(d) == r.idx;
            } else {
              const double uq = static_cast<double>(u) * qd, e = exp(x);
              const double off = r.s * a.sum_error;
              pass = uq * (r.s + off) < e ? 1 : (uq * (r.s - off) < e ? kPassOpen : 0);
              s_uq[warp] = uq;
            }
          }
          s_pass[warp] = valid || i == n ? pass : -1;
          s_x[warp] = x;
          s_rows[warp] = r;
        }
      }
      __syncthreads();
      for (int w = 0; w < kVfyWarps && i0 + w <= n; ++w) {
        int pass = s_pass[w];
        if (pass == kPassOpen) {  // too close to the border for a sum in 32 bits
          const double sum = row_sum_f64<T>(a, logits + (row0 + i0 + w) * a.ld_logits, s_rows[w].m, st.t, s_exp2, s_lane,
                                            s_warp);
          pass = s_uq[w] * sum < exp(s_x[w]);
        }
        if (pass != 1) {
          acc = i0 + w;
          break;
        }
      }
      const int64_t upto = acc < 0 ? i0 + kVfyWarps : acc;
      if (threadIdx.x < kVfyWarps && i0 + threadIdx.x < upto) {
        a.tokens[row0 + i0 + threadIdx.x] = __ldg(a.drafts + lo + i0 + threadIdx.x);
        a.log_probs[row0 + i0 + threadIdx.x] =
            static_cast<float>(s_x[threadIdx.x] - log(static_cast<double>(s_rows[threadIdx.x].s)));
      }
      if (acc >= 0 && threadIdx.x == 0) {
        const RowStats r = s_rows[acc - i0];
        s_decision = {acc, r.m, r.s};
        if (s_pass[acc - i0] < 0 && a.status != nullptr) atomicOr(a.status, kStatusBadTarget);
        a.accepted[b] = acc;
        // Nothing to draw, or what the draw's own CTA writes over after the cluster's next barrier: should no warp
        // take the number, which only logits written during the call could cause, the row is defined all the same.
        const bool none = r.s == 0.0f || !st.greedy;
        a.tokens[row0 + acc] = none ? -1 : static_cast<int64_t>(r.idx);
        a.log_probs[row0 + acc] = none ? -INFINITY : static_cast<float>(-log(static_cast<double>(r.s)));
      }
      __syncthreads();
    }
    const int64_t last = b == a.batch - 1 ? a.n_drafts + a.batch - 1 : row0 + n;
    for (int64_t i = row0 + acc + 1 + threadIdx.x; i <= last; i += kVfyThreads) {
      a.tokens[i] = -1;
      a.log_probs[i] = 0.0f;
    }
    if (b == 0) {
      for (int64_t i = threadIdx.x; i < row0; i += kVfyThreads) {
        a.tokens[i] = -1;
        a.log_probs[i] = 0.0f;
      }
    }
  }
  cluster_sync_all();
  const Decision decision = ld_cluster_decision(&s_decision, 0);
  const int64_t acc = decision.acc, row = row0 + acc;
  const RowStats rs = {decision.m, decision.s, 0};
  if (rs.s == 0.0f || st.greedy) {
    cluster_sync_all();  // the first CTA stays until all have read its decision
    return;
  }

  // ---- draw from row `row`
  DrawRow d = draw_row(logits + row * a.ld_logits, rs.m, st.t);
  d.q = a.q == nullptr ? nullptr : static_cast<const Q*>(a.q) + (lo + acc) * a.ld_q;
  // columns of this CTA, and of each of its warps, in order, in groups of strip_step strips of 256
  const int group_cols = 256 * a.strip_step;
  const int warps = static_cast<int>(ctas) * kVfyWarps;
  const int64_t per_warp = ((a.vocab + warps - 1) / warps + group_cols - 1) / group_cols * group_cols;
  const int w_lo = static_cast<int>(min(a.vocab, (static_cast<int64_t>(rank) * kVfyWarps + warp) * per_warp));
  const int w_hi = static_cast<int>(min(a.vocab, w_lo + per_warp));
  int exchange = 0;
  double total = 0.0, before = 0.0, mine = 0.0, theirs = 0.0;
  // This warp's sum of weights (mine), the sum of all columns before this CTA's (before) and of all
  // columns (total); the lanes' sums of each group stay in s_lane.
  auto sum_weights = [&]() {
    mine = d.mode == kDrawResidual ? sum_columns<T, Q, true>(a, d, s_exp2, w_lo, w_hi, group_cols, s_lane)
                                   : sum_columns<T, Q, false>(a, d, s_exp2, w_lo, w_hi, group_cols, s_lane);
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
    // lane k reads CTA k's sum, so that the reads are in flight together
    theirs = static_cast<uint32_t>(lane) < ctas ? ld_cluster_f64(&s_total[exchange], lane) : 0.0;
    total = before = 0.0;
    for (uint32_t k = 0; k < ctas; ++k) {
      const double t = __shfl_sync(0xffffffffu, theirs, static_cast<int>(k));
      if (k < rank) before += t;
      total += t;
    }
    exchange ^= 1;
  };
  // One copy of the pass, so that its code stays in the instruction cache: with draft probabilities first the
  // softmax denominator in 64 bits, then the weights, and p when nothing is left of those.
  bool denominator = false;
  if (acc < n) {
    denominator = a.q != nullptr;
    if (!denominator) {
      d.mode = kDrawWithout;
      const int64_t t = __ldg(a.drafts + lo + acc);
      d.without = t >= 0 && t < a.vocab ? static_cast<int>(t) : -1;
    }
  }
#pragma unroll 1
  for (;;) {
    sum_weights();
    if (denominator) {
      denominator = false;
      // every CTA has passed the exchange, so this one's warps are done with the table
      const double inv = 1.0 / total;
      for (int j = threadIdx.x; j < kExp2Entries; j += kVfyThreads) s_exp2[j] *= inv;
      __syncthreads();
      d.mode = kDrawResidual;
    } else if (total > 0.0 || d.mode == kDrawP) {
      break;
    } else {
      d.mode = kDrawP;
      d.without = -1;
    }
  }
  // x = r * total falls to the last warp with any weight whose columns start at or before x (so exactly
  // one takes it, whatever rounding does at the ends).
  const float rf = __ldg(a.final_uniforms + b);
  const double x = (rf >= 0.0f ? fmin(static_cast<double>(rf), 1.0) : 0.0) * total;
  // where the next CTA's columns start, and whether a later CTA has weight
  const double after = before + __shfl_sync(0xffffffffu, theirs, static_cast<int>(rank));
  const bool later = __any_sync(0xffffffffu, static_cast<uint32_t>(lane) > rank && theirs > 0.0);
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
    // The last group with any weight that starts at or before x, from the kept sums; then its strips.
    // lane g: the sum of group g, and of those before it
    double group_sum = 0.0;
    const int groups = (w_hi - w_lo + group_cols - 1) / group_cols;
#pragma unroll 4
    for (int g = 0; g < groups; ++g) {
      const double sum = warp_sum(s_lane[g][threadIdx.x]);
      if (lane == g) group_sum = sum;
    }
    double upto = group_sum;
#pragma unroll
    for (int o = 1; o < kVfyMaxGroups; o <<= 1) {
      const double t = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += t;
    }
    double run = fmax(start + (upto - group_sum), start);
    const uint32_t starts = __ballot_sync(0xffffffffu, group_sum > 0.0 && run <= x);
    const int g = starts != 0 ? 31 - __clz(starts) : 0;  // the first live group starts at `start`, so there is one
    run = __shfl_sync(0xffffffffu, run, g);
    const int at = w_lo + g * group_cols;
    const int g1 = min(w_hi, at + group_cols);
    int token = -1, last_live = -1;
#pragma unroll 1
    for (int c0 = at; c0 < g1 && token < 0; c0 += 256) {
      const int c = c0 + lane * 8;
      const T* zp = static_cast<const T*>(d.z) + c;
      const Q* qp = static_cast<const Q*>(d.q) + c;
      double w[8];
      bool is_live[8];
      if (d.mode == kDrawResidual) {
        DrawCols<T, Q, true> cols;
        cols.load(zp, qp, 1, g1 - c, a.logits_vec != 0 && a.q_vec != 0);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          w[j] = draw_weight<T, Q, true>(d, s_exp2, cols.z.at(j), cols.q.at(j), is_live[j]);
          is_live[j] = is_live[j] && w[j] > 0.0;
        }
      } else {
        DrawCols<T, Q, false> cols;
        cols.load(zp, qp, 1, g1 - c, a.logits_vec != 0);
        mask_without(d, cols.z, c, 1);
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = draw_weight<T, Q, false>(d, s_exp2, cols.z.at(j), 0.0f, is_live[j]);
      }
      double sum = 0.0;
      int live = -1;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (is_live[j]) {
          sum += w[j];
          live = j;
        }
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
        if (is_live[j]) {
          cur += w[j];
          if (hit < 0 && cur > x) hit = j;
        }
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
    if (token < 0) token = last_live;  // what rounding leaves past the end
    // The sums say that this group has a live column. Logits that another stream is still writing while they are read
    // may have none left by now: the token is then -1, and nothing is read before the row.
    if (lane == 0) {
      a.tokens[row] = token;
      double logp = -INFINITY;
      if (token >= 0) {
        const double z = clean_logit<T>(to_f32<T>(static_cast<const T*>(d.z)[token]));
        logp = (z - rs.m) / st.t - log(static_cast<double>(rs.s));
      }
      a.log_probs[row] = static_cast<float>(logp);
    }
  }
  cluster_sync_all();  // no CTA leaves while another may still read its sums
}

// CTAs per sequence: many for few sequences, whose columns they share; fewer when the batch fills the GPU anyway,
// since each CTA of a cluster waits for the decision. Three CTAs fit an SM. A batch that draws in every sequence is fastest
// when all its clusters are resident together; greedy sequences leave early, so that a batch of mixed temperatures is
// faster with up to 4 per SM. A temperature for all tells the two apart, temperatures of each do not. us with 8, 4, 2 and 1
// CTAs, logits in bf16, 4 drafts per sequence (0 to 7 drafts: the same best ones, but 2 for 128 with probabilities at V = 128256):
//                  V = 32000                                    V = 128256
//   sequences      with draft probabilities    without          with draft probabilities      without
//   32             20, 20, 24, 32              16, 16, 18, 21   37, 40, 54, 83                28, 29, 34, 46
//   64             34, 27, 29, 37              29, 19, 20, 23   67, 61, 67, 91                51, 42, 45, 55
//   96             44, 33, 35, 38              34, 24, 25, 26   88, 79, 89, 104               65, 56, 60, 69
//   128            57, 45, 36, 40              46, 37, 27, 28   113, 105, 117, 133            86, 83, 77, 82
//   192            80, 56, 48, 54              63, 44, 36, 38   160, 139, 135, 157            122, 102, 93, 102
//   256            105, 75, 66, 61             87, 61, 52, 44   218, 191, 182, 183            171, 146, 134, 127
//   512            204, 138, 114, 111          168, 111, 91, 85 396, 329, 300, 314            304, 245, 213, 217
// A quarter of the sequences greedy: 64 of 0 to 7 drafts, V = 128256, fp32 probabilities 55, 58, 62, 92; 256 of 4, V = 32000,
// fp32 logits, bf16 probabilities 104, 76, 67, 73.
inline int verify_cluster(int64_t batch, int64_t vocab, int sms, bool all_draw) {
  const int limit = (all_draw ? 3 : 4) * sms;
  int ctas = kVfyMaxCluster;
  while (ctas > 1 && (batch * ctas > limit || vocab <= 256 * kVfyWarps * (ctas / 2))) ctas /= 2;
  return ctas;
}

template <typename T, typename Q>
static int launch_verify(VerifyArgs& a, cudaStream_t stream) {
  int sms = 0;
  int rc = sm_count(&sms);
  if (rc) return rc;
  const int ctas = verify_cluster(a.batch, a.vocab, sms, a.temperature == nullptr && a.temperature_all >= kVfyMinTemp);
  FRX_REQUIRE(a.batch * ctas < (1ll << 31), FRX_ERR_INVALID_ARG, "frx_verify_drafts: too many sequences (%lld)",
              (long long)a.batch);
  // a warp's columns in at most kVfyMaxGroups groups
  const int64_t strips = (a.vocab + 256ll * ctas * kVfyWarps - 1) / (256ll * ctas * kVfyWarps);
  a.strip_step = static_cast<int>((strips + kVfyMaxGroups - 1) / kVfyMaxGroups);
  // Longer chunks spare a warp's set-up and its joins, as long as they leave the GPU 32 warps per SM.
  a.chunk_cols = kVfyChunk;
  const int64_t rows = a.n_drafts + a.batch;
  while (a.chunk_cols < 16 * kVfyChunk && rows * ((a.vocab + 2 * a.chunk_cols - 1) / (2 * a.chunk_cols)) >= 32ll * sms)
    a.chunk_cols *= 2;
  a.n_chunks = static_cast<int>((a.vocab + 7 + a.chunk_cols - 1) / a.chunk_cols);
  a.sum_error = stats_sum_error(a.n_chunks);
  const int64_t mean_rows = (a.n_drafts + 2 * a.batch - 1) / a.batch;
  a.row_step = static_cast<int>(mean_rows < 64 ? mean_rows : 64);
  const dim3 grid(static_cast<unsigned>((a.n_chunks + kVfyWarps - 1) / kVfyWarps),
                  static_cast<unsigned>(a.batch < 65535 ? a.batch : 65535), static_cast<unsigned>(a.row_step));
  // The sample kernel's clusters are placed where there is room. Beside a statistics kernel that fills most SMs they
  // would share the few others (8 sequences, V = 128256: 32 us instead of 26); beside a small one they start earlier
  // (1 sequence: 20.6 us instead of 21.9).
  a.early = static_cast<int64_t>(grid.x) * grid.y * grid.z + a.batch * ctas <= 2 * sms;
  verify_stats_kernel<T><<<grid, kVfyThreads, 0, stream>>>(a);
  FRX_CUDA_CHECK(cudaGetLastError());
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.batch * ctas), 1, 1);
  cfg.blockDim = dim3(kVfyThreads, 1, 1);
  cfg.dynamicSmemBytes = 0;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(ctas);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  FRX_CUDA_CHECK(cudaLaunchKernelEx(&cfg, verify_sample_kernel<T, Q>, static_cast<const VerifyArgs>(a)));
  return FRX_OK;
}

template <typename T>
static int launch_verify_q(VerifyArgs& a, int q_dtype, cudaStream_t stream) {
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
  FRX_REQUIRE(batch >= 0 && n_drafts >= 0 && vocab >= 1 && vocab < (1ll << 30) && batch < (1ll << 31) &&
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
  const int64_t n_chunks = (vocab + 7 + kVfyChunk - 1) / kVfyChunk;
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
  static const Exp2Table exp2 = make_exp2_table();
  VerifyArgs a = {};
  a.exp2 = exp2;
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
