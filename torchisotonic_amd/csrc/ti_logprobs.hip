// Log-probabilities of given tokens under a language model's logits, with the entropy of each row's
// distribution, and their gradient.
//
// For a row z of `vocab` logits, a target t and a temperature T, with m = max z,
//
//   s = sum_j exp((z_j - m) / T),      logp = (z_t - m) / T - log s,
//   q = sum_j exp((z_j - m) / T) (z_j - m) / T,      H = log s - q / s,
//
// and for the upstream gradients g of logp and gH of H, with p_j = exp((z_j - m) / T) / s,
//
//   dz_j = (g ((j == t) - p_j) - gH p_j (log p_j + H)) / T.
//
// The forward keeps m and s of every row; the backward reads the logits once more and forms p from
// them. A row whose target is the ignored one gives zeros and is not read; a target outside the
// vocabulary gives NaN, in the row's gradient too. A logit of -inf is a token of probability zero,
// whose p (log p) is zero; a row of nothing else has no distribution and gives NaN, as a row that
// holds a NaN or +inf does.
#include <hip/hip_runtime.h>

#include <cmath>
#include <type_traits>

#include "ti_common.h"
#include "ti_kernels.h"

namespace ti {

namespace {

constexpr int kThreads = 256;

template <typename T>
struct AccOf {
  using type = float;
};
template <>
struct AccOf<double> {
  using type = double;
};

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ double exp2_of(double x) { return exp2(x); }
__device__ __forceinline__ float max_of(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double max_of(double a, double b) { return fmax(a, b); }
__device__ __forceinline__ float fma_of(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fma_of(double a, double b, double c) { return __builtin_fma(a, b, c); }

// Up to `near` the rounding of a logit times log2(e) / T is at most half a binade; `lowest` stands in for an
// exponent of -inf: its power is zero, as that of every exponent below it is.
template <typename A>
struct Limits;
template <>
struct Limits<float> {
  static constexpr float near = 0x1p24f, lowest = -1.0e4f, largest = 3.402823466e38f;
};
template <>
struct Limits<double> {
  static constexpr double near = 0x1p53, lowest = -1.0e4, largest = 1.7976931348623157e308;
};

// log2(e) / T and 1 / T in the type of the sums; the largest finite value where T is too small for them (what is
// not a row's largest logit has probability zero long before).
template <typename A>
__device__ __forceinline__ A per_temperature(double x, double temperature) {
  const double v = x / temperature;
  return v < static_cast<double>(Limits<A>::largest) ? static_cast<A>(v) : Limits<A>::largest;
}
template <typename A>
__device__ __forceinline__ A log2e_over(double temperature) {
  return per_temperature<A>(1.4426950408889634074, temperature);
}

// x, or a finite stand-in for -inf. (For a NaN too: the exponential that it goes with is NaN.)
template <typename A>
__device__ __forceinline__ A above_lowest(A x) {
  return max_of(x, Limits<A>::lowest);
}

// The exponent of a logit z against the largest known one, m: with c = log2(e) / T and b = m c as
// rounded, z c - b in one operation, rounded once (4.5 instructions an element where z - m and a product
// made 5.5). b is only a point of reference: what its rounding moved it by, `excess`, is in every exponent
// of the row alike and leaves the log of the sum again. That holds while it is small: past `near`, as in a
// row masked whole with a large finite value or at a small temperature, it would take the powers out of
// their range (by 2^440 where m c is -1.4e10), and the exponents are (z - m) c.
template <typename A>
struct Scale {
  A c, m, b;
  bool plain;
  __device__ __forceinline__ Scale(A m_, A c_) : c(c_), m(m_ == A(-INFINITY) ? A(0) : m_) {
#pragma clang fp contract(off)
    b = m * c;
    plain = b >= -Limits<A>::near && b <= Limits<A>::near;
  }
  // What the exponents are above their exact values, in all of a row's alike.
  __device__ __forceinline__ A excess() const { return plain ? fma_of(m, c, -b) : A(0); }
};

// What is known of some of a row's logits: their largest, the sum of exp2 of their exponents against it,
// and (ENT) the sum of those times the exponents. (The largest leaves NaN out; its exponential makes the
// sum NaN.)
template <typename A, bool ENT>
struct Part {
  A m = A(-INFINITY), s = A(0), q = A(0);

  // The sums against a larger m, whose scale is `to`. Their own point of reference is m c as rounded where that
  // is near, else m c as it is, whatever the larger one's.
  __device__ __forceinline__ void move(A larger, const Scale<A>& to) {
    // (no contraction of m c with the difference)
#pragma clang fp contract(off)
    const A own = m * to.c;
    const A over = own >= -Limits<A>::near && own <= Limits<A>::near ? fma_of(m, to.c, -own) : A(0);
    const A d = (to.plain ? fma_of(m, to.c, -to.b) : (m - to.m) * to.c) - over, f = exp2_of(d);
    if constexpr (ENT) q = f * (q + s * above_lowest(d));
    s *= f;
    m = larger;
  }

  template <int K>
  __device__ __forceinline__ void add(const A (&z)[K], A c) {
    A top = z[0];
#pragma unroll
    for (int i = 1; i < K; ++i) top = max_of(top, z[i]);
    const A larger = max_of(m, top);
    const Scale<A> scale(larger, c);
    move(larger, scale);
    if (scale.plain) add_all(z, [&](A v) { return fma_of(v, c, -scale.b); });
    else add_all(z, [&](A v) { return (v - scale.m) * c; });
  }

  // (four sums side by side: chains of additions a quarter as long)
  template <int K, typename Exponent>
  __device__ __forceinline__ void add_all(const A (&z)[K], Exponent exponent) {
    constexpr int kSums = K < 4 ? K : 4;
    A e4[kSums], q4[kSums];
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const A x = exponent(z[i]), e = exp2_of(x);
      e4[i % kSums] = i < kSums ? e : e4[i % kSums] + e;
      if constexpr (ENT) q4[i % kSums] = i < kSums ? e * above_lowest(x) : fma_of(e, above_lowest(x), q4[i % kSums]);
    }
#pragma unroll
    for (int d = 1; d < kSums; d *= 2)
#pragma unroll
      for (int i = 0; i + d < kSums; i += 2 * d) {
        e4[i] += e4[i + d];
        if constexpr (ENT) q4[i] += q4[i + d];
      }
    s += e4[0];
    if constexpr (ENT) q += q4[0];
  }

};

struct Rows {
  int64_t inner, outer_stride, row_stride;  // row r begins at (r / inner) * outer_stride + (r % inner) * row_stride
  __device__ __forceinline__ int64_t at(int64_t r) const {
    if (r < inner) return r * row_stride;
    const int64_t o = r / inner;
    return o * outer_stride + (r - o * inner) * row_stride;
  }
};

// 16 bytes of a row, at any alignment of an element's.
template <typename T>
struct Vec {
  static constexpr int kN = 16 / sizeof(T);
  using type = T __attribute__((ext_vector_type(kN)));
};

template <typename T>
__device__ __forceinline__ typename Vec<T>::type load16(const T* p) {
  typename Vec<T>::type v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
// Past the caches, for the backward: its gradient is read by later kernels, and its logits by none, so
// that what the forward left in the last-level cache (256 MB) stays there until the backward reads it.
// 8192 x 128000 bfloat16, forward and backward: 1010 us, with ordinary loads 1098 us; 4096 x 32000 float32
// with entropy 236 and 255 us, and with ordinary stores too about 60 us more.
template <typename T>
using Unaligned16 = T __attribute__((ext_vector_type(Vec<T>::kN), aligned(sizeof(T))));
template <typename T>
__device__ __forceinline__ typename Vec<T>::type load16_last(const T* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const Unaligned16<T>*>(p));
}
template <typename T>
__device__ __forceinline__ void store16(T* p, typename Vec<T>::type v) {
  __builtin_nontemporal_store(v, reinterpret_cast<Unaligned16<T>*>(p));
}

// A row of at least kN elements as 16-byte vectors: vector 0 at its start, the others from the first
// 16-byte boundary of `base` on, the last one moved back to end with the row. Vectors 2 to count - 2
// neither overlap nor leave the row.
template <typename T>
struct Vectors {
  static constexpr int kN = Vec<T>::kN;
  int first, vocab, count;
  __device__ __forceinline__ Vectors(const T* base, int n) : vocab(n) {
    const int to_line = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(base) & 15)) & 15) / static_cast<int>(sizeof(T));
    first = to_line == 0 ? kN : to_line;
    count = 1 + (n - first + kN - 1) / kN;
  }
  __device__ __forceinline__ int unmoved(int k) const { return k == 0 ? 0 : first + (k - 1) * kN; }
  __device__ __forceinline__ int start(int k) const {
    const int at = unmoved(k);
    return at < vocab - kN ? at : vocab - kN;
  }
  // The first of the vector's elements that no vector before it holds.
  __device__ __forceinline__ int fresh(int k) const { return k == 1 ? kN : unmoved(k); }
};

// The results of row r from its sums, by one lane; zt: the target's logit.
template <typename A, bool ENT>
struct Results {
  A *logp, *entropy;
  A* stats;  // null: no backward follows
  int64_t rows;
  __device__ __forceinline__ void put(int64_t r, const Part<A, ENT>& p, A zt, double temperature) const {
    constexpr A kLn2 = static_cast<A>(0.69314718055994530942);
    const Scale<A> scale(p.m, log2e_over<A>(temperature));
    const A logs = log(p.s);
    logp[r] = (zt - p.m) * per_temperature<A>(1.0, temperature) - (logs - scale.excess() * kLn2);
    if constexpr (ENT) entropy[r] = logs - p.q / p.s * kLn2;
    keep(r, p.m, p.s);
  }
  __device__ __forceinline__ void put_ignored(int64_t r) const {
    logp[r] = A(0);
    if constexpr (ENT) entropy[r] = A(0);
    keep(r, A(0), A(1));
  }
  __device__ __forceinline__ void keep(int64_t r, A m, A s) const {
    if (stats == nullptr) return;
    stats[r] = m;
    stats[rows + r] = s;
  }
};

template <typename T>
__device__ __forceinline__ typename AccOf<T>::type at_target(const T* z, int64_t t, int vocab) {
  using A = typename AccOf<T>::type;
  return t >= 0 && t < vocab ? static_cast<A>(z[t]) : quiet_nan<A>();
}

// The value of the lane that DPP control CTRL names, of the same 16 lanes.
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __builtin_bit_cast(float, dpp_i32<CTRL, 0xF>(__builtin_bit_cast(int, x)));
}
template <int CTRL>
__device__ __forceinline__ double dpp(double x) {
  return dpp_f64<CTRL, 0xF>(x);
}
// The sum, or the largest, over the G lanes of a group (4 at least), in each of them: with the neighbour, the
// other pair, then the mirrored lane of 8 and of 16 (whose quads, then halves, hold one value each).
template <int G, typename A, typename Op>
__device__ __forceinline__ A over_group(A x, Op op) {
  x = op(x, dpp<0xB1>(x));   // quad_perm 1 0 3 2
  x = op(x, dpp<0x4E>(x));   // quad_perm 2 3 0 1
  if constexpr (G > 4) x = op(x, dpp<0x141>(x));  // row_half_mirror
  if constexpr (G > 8) x = op(x, dpp<0x140>(x));  // row_mirror
  if constexpr (G > 16) x = op(x, __shfl_xor(x, 16));
  if constexpr (G > 32) x = op(x, __shfl_xor(x, 32));
  return x;
}

// Bound by its vector instructions and the latency of a wave's few loads: 65536 rows of 257 float16 (34 MB)
// in 9.1 us, 3.8 TB/s; 32768 of 2000 bfloat16 (131 MB) in 25 us, 5.2 TB/s. (With a running maximum and
// joins across the lanes, as the long rows have, 13.2 and 33 us.)
//
// Short rows, G lanes each, whole in registers: U vectors a lane and the elements past the last whole
// vector one a lane, so that the row's largest is known before the first exponential.
template <typename T, bool ENT, int G, int U>
__global__ __launch_bounds__(kThreads) void logprobs_short_kernel(const T* __restrict__ logits,
                                                                  const int64_t* __restrict__ targets,
                                                                  Results<typename AccOf<T>::type, ENT> out, int vocab,
                                                                  Rows where, int64_t ignore, double temperature) {
  using A = typename AccOf<T>::type;
  constexpr int kN = Vec<T>::kN;
  const int lane = threadIdx.x % G;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * (kThreads / G) + threadIdx.x / G;
  const bool some = r < out.rows;
  const int64_t t = some ? targets[r] : ignore;
  const bool kept = t != ignore;
  const A c = log2e_over<A>(temperature);
  const T* z = logits + (kept ? where.at(r) : 0);
  const int whole = vocab / kN;
  typename Vec<T>::type v[U];
  A rest = A(-INFINITY), zt = A(0);
#pragma unroll
  for (int u = 0; u < U; ++u) {
#pragma unroll
    for (int i = 0; i < kN; ++i) v[u][i] = static_cast<T>(-INFINITY);
    if (kept && lane + u * G < whole) v[u] = load16(z + static_cast<int64_t>(lane + u * G) * kN);
  }
  if (kept) {
    if (lane < vocab - whole * kN) rest = static_cast<A>(z[whole * kN + lane]);
    if (lane == 0) zt = at_target(z, t, vocab);
  }
  Part<A, ENT> p;
  A top = rest;
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (u * G < whole) {
#pragma unroll
      for (int i = 0; i < kN; ++i) top = max_of(top, static_cast<A>(v[u][i]));
    }
  p.m = over_group<G>(top, [](A a, A b) { return max_of(a, b); });
  const Scale<A> scale(p.m, c);
  A s[4] = {A(0), A(0), A(0), A(0)}, q[4] = {A(0), A(0), A(0), A(0)};
  auto add_row = [&](auto exponent) {
    auto add = [&](A z1, int i) {
      const A x = exponent(z1), e = exp2_of(x);
      s[i] += e;
      if constexpr (ENT) q[i] = fma_of(e, above_lowest(x), q[i]);
    };
    add(rest, 0);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u * G < whole) {
#pragma unroll
        for (int i = 0; i < kN; ++i) add(static_cast<A>(v[u][i]), i % 4);
      }
  };
  if (scale.plain) add_row([&](A z1) { return fma_of(z1, c, -scale.b); });
  else add_row([&](A z1) { return (z1 - scale.m) * c; });
  auto plus = [](A a, A b) { return a + b; };
  p.s = over_group<G>((s[0] + s[1]) + (s[2] + s[3]), plus);
  if constexpr (ENT) p.q = over_group<G>((q[0] + q[1]) + (q[2] + q[3]), plus);
  if (lane != 0 || !some) return;
  if (kept) out.put(r, p, zt, temperature);
  else out.put_ignored(r);
}

// The parts of a group of G lanes joined, in each of them: moved to the largest of all, then summed.
template <int G, typename A, bool ENT>
__device__ __forceinline__ void join_group(Part<A, ENT>& p, A c) {
  auto plus = [](A a, A b) { return a + b; };
  const A larger = over_group<G>(p.m, [](A a, A b) { return max_of(a, b); });
  p.move(larger, Scale<A>(larger, c));
  p.s = over_group<G>(p.s, plus);
  if constexpr (ENT) p.q = over_group<G>(p.q, plus);
}

// The parts of each wave's 64 lanes, then of the workgroup's waves.
template <int NT, typename A, bool ENT>
__device__ __forceinline__ void join_all(Part<A, ENT>& p, A c) {
  join_group<64>(p, c);
  if constexpr (NT > 64) {
    constexpr int kWaves = NT / 64;
    __shared__ A parts[3][kWaves];
    const int wave = threadIdx.x / 64;
    if (threadIdx.x % 64 == 0) {
      parts[0][wave] = p.m;
      parts[1][wave] = p.s;
      if constexpr (ENT) parts[2][wave] = p.q;
    }
    __syncthreads();
    p.m = parts[0][threadIdx.x % kWaves];
    p.s = parts[1][threadIdx.x % kWaves];
    if constexpr (ENT) p.q = parts[2][threadIdx.x % kWaves];
    join_group<kWaves>(p, c);
  }
}

// Bound by its reads: 8192 rows of 128000 bfloat16 (2.1 GB) in 329 us, 6.4 TB/s, above a copy's rate; 256
// rows, one a compute unit, in 15.1 us, 4.3 TB/s, of which the exponentials' instructions are about 7 us.
//
// Long rows, NT threads each (rows of at least three vectors). With `parts`, workgroup (r, y) takes the
// y-th of gridDim.y stretches of the row and leaves its sums there.
template <typename T, bool ENT, int NT>
__global__ __launch_bounds__(NT) void logprobs_kernel(const T* __restrict__ logits, const int64_t* __restrict__ targets,
                                                      Results<typename AccOf<T>::type, ENT> out, int vocab, Rows where,
                                                      int64_t ignore, double temperature,
                                                      Part<typename AccOf<T>::type, ENT>* __restrict__ parts) {
  using A = typename AccOf<T>::type;
  constexpr int kN = Vec<T>::kN, U = 4;
  const int64_t r = blockIdx.x;
  const int64_t t = targets[r];
  if (t == ignore) {
    if (threadIdx.x == 0 && blockIdx.y == 0) out.put_ignored(r);
    return;
  }
  const A c = log2e_over<A>(temperature);
  const T* z = logits + where.at(r);
  const A zt = threadIdx.x == 0 ? at_target(z, t, vocab) : A(0);
  Part<A, ENT> p;
  const Vectors<T> vs(z, vocab);
  if (threadIdx.x < 3 && blockIdx.y == 0) {
    const int k = threadIdx.x < 2 ? threadIdx.x : vs.count - 1;
    const typename Vec<T>::type v = load16(z + vs.start(k));
    const int dead = vs.fresh(k) - vs.start(k);
    A x[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) x[i] = i < dead ? A(-INFINITY) : static_cast<A>(v[i]);
    p.add(x, c);
  }
  const T* from = z + vs.first + kN;  // vector 2
  const int n = vs.count - 3;
  const int each = (n + gridDim.y - 1) / gridDim.y, begin = blockIdx.y * each;
  const int end = begin + each < n ? begin + each : n;
  int k = begin + threadIdx.x;
  for (; k + (U - 1) * NT < end; k += U * NT) {
    typename Vec<T>::type v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load16(from + static_cast<int64_t>(k + u * NT) * kN);
    A x[U * kN];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < kN; ++i) x[u * kN + i] = static_cast<A>(v[u][i]);
    p.add(x, c);
  }
  for (; k < end; k += NT) {
    const typename Vec<T>::type v = load16(from + static_cast<int64_t>(k) * kN);
    A x[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) x[i] = static_cast<A>(v[i]);
    p.add(x, c);
  }
  join_all<NT>(p, c);
  if (threadIdx.x != 0) return;
  if (parts != nullptr) parts[r * gridDim.y + blockIdx.y] = p;
  else out.put(r, p, zt, temperature);
}

// A row's stretches (at most 64) joined, a wave a row.
template <typename T, bool ENT>
__global__ __launch_bounds__(64) void logprobs_join_kernel(const T* __restrict__ logits,
                                                           const int64_t* __restrict__ targets,
                                                           Results<typename AccOf<T>::type, ENT> out, int vocab,
                                                           Rows where, int64_t ignore, double temperature,
                                                           const Part<typename AccOf<T>::type, ENT>* __restrict__ parts,
                                                           int count) {
  using A = typename AccOf<T>::type;
  const int64_t r = blockIdx.x;
  const int64_t t = targets[r];
  if (t == ignore) return;
  const A c = log2e_over<A>(temperature);
  Part<A, ENT> p;
  if (static_cast<int>(threadIdx.x) < count) p = parts[r * count + threadIdx.x];
  const A zt = threadIdx.x == 0 ? at_target(logits + where.at(r), t, vocab) : A(0);
  join_all<64>(p, c);
  if (threadIdx.x == 0) out.put(r, p, zt, temperature);
}

// Bound by its reads and writes: 8192 rows of 128000 bfloat16 (4.2 GB) in 695 us alone, 6.0 TB/s, and 677 us
// after its forward.
//
// G lanes a row; where G is the workgroup, `chunks` workgroups a row, each up to kGradVectors * G vectors.
constexpr int kGradVectors = 4;

template <typename T, bool ENT, int G>
__global__ __launch_bounds__(kThreads) void logprobs_grad_kernel(
    const T* __restrict__ logits, const int64_t* __restrict__ targets, const typename AccOf<T>::type* __restrict__ stats,
    const typename AccOf<T>::type* __restrict__ entropy, const typename AccOf<T>::type* __restrict__ g,
    const typename AccOf<T>::type* __restrict__ ge, T* __restrict__ grad, int64_t rows, int vocab, Rows where,
    int64_t ignore, double temperature, unsigned chunks, bool mixed) {
  using A = typename AccOf<T>::type;
  constexpr int kN = Vec<T>::kN;
  const int lane = threadIdx.x % G;
  // (a row's chunks one after another, so that what is read and written together lies together: chunk by
  // chunk over all rows took 822 us where this takes 695 us, 8192 rows of 128000 bfloat16)
  const unsigned chunk = G >= kThreads ? blockIdx.x % chunks : 0;
  unsigned block = G >= kThreads ? blockIdx.x / chunks : blockIdx.x;
  // (rows from both ends in turn: the forward's last ones are still in the last-level cache)
  if (mixed) block = block % 2 == 0 ? gridDim.x / chunks - 1 - block / 2 : block / 2;
  const int64_t r = static_cast<int64_t>(block) * (kThreads / G) + threadIdx.x / G;
  if (r >= rows) return;
  const int64_t target = targets[r];
  T* out = grad + r * vocab;
  const bool kept = target != ignore, in = target >= 0 && target < vocab;
  const int t = in ? static_cast<int>(target) : -kN;
  const T* z = logits + (kept ? where.at(r) : 0);
  const A c = log2e_over<A>(temperature), inv = per_temperature<A>(1.0, temperature);
  const Scale<A> scale(stats[r], c);
  const A s = stats[rows + r];
  const A gr = !in ? quiet_nan<A>() : (g != nullptr ? g[r] * inv : A(0));
  // d_j = e_j a + (e_j x_j) b, and gr more at the target (e_j x_j first: zero times a large b)
  A a = -gr / s, b = A(0);
  if constexpr (ENT) {
    const A gh = ge[r] * inv;
    a -= gh * (entropy[r] - log(s)) / s;
    b = -gh * static_cast<A>(0.69314718055994530942) / s;
  }
  auto of = [&](A x) {
    const A e = exp2_of(x);
    return ENT ? fma_of(e * above_lowest(x), b, e * a) : e * a;
  };
  auto of_one = [&](A v) { return of(scale.plain ? fma_of(v, c, -scale.b) : (v - scale.m) * c); };
  auto put = [&](int start, typename Vec<T>::type v) {
    A d[kN];
    if (scale.plain) {
#pragma unroll
      for (int i = 0; i < kN; ++i) d[i] = of(fma_of(static_cast<A>(v[i]), c, -scale.b));
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i) d[i] = of((static_cast<A>(v[i]) - scale.m) * c);
    }
    if (t >= start && t < start + kN) {
#pragma unroll
      for (int i = 0; i < kN; ++i) d[i] += start + i == t ? gr : A(0);
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = static_cast<T>(d[i]);
    store16(out + start, v);
  };
  const typename Vec<T>::type zero = {};
  typename Vec<T>::type v[kGradVectors];
  if constexpr (G >= kThreads) {
    // (even shares of the row: 16384 rows of 9000 in two of 2.2 vectors a thread, 109 us, where 4 and 0.4
    // took 119 us; an element that two vectors hold gets the same value from both)
    const Vectors<T> vs(out, vocab);
    const int each = (vs.count + chunks - 1) / chunks;
    const int k0 = chunk * each + lane;
    const int end = k0 - lane + each < vs.count ? k0 - lane + each : vs.count;
#pragma unroll
    for (int u = 0; u < kGradVectors; ++u)
      if (kept && k0 + u * G < end) v[u] = load16_last(z + vs.start(k0 + u * G));
#pragma unroll
    for (int u = 0; u < kGradVectors; ++u)
      if (k0 + u * G < end) {
        if (kept) put(vs.start(k0 + u * G), v[u]);
        else store16(out + vs.start(k0 + u * G), zero);
      }
  } else {
    const int whole = vocab / kN, rest = whole * kN + lane;
    const A z1 = kept && rest < vocab ? static_cast<A>(z[rest]) : A(0);
    for (int k0 = lane; k0 < whole; k0 += kGradVectors * G) {
#pragma unroll
      for (int u = 0; u < kGradVectors; ++u)
        if (kept && k0 + u * G < whole) v[u] = load16_last(z + (k0 + u * G) * kN);
#pragma unroll
      for (int u = 0; u < kGradVectors; ++u)
        if (k0 + u * G < whole) {
          if (kept) put((k0 + u * G) * kN, v[u]);
          else store16(out + (k0 + u * G) * kN, zero);
        }
    }
    if (rest < vocab) out[rest] = kept ? static_cast<T>(of_one(z1) + (rest == t ? gr : A(0))) : T(0);
  }
}

// Lanes a row of at most kShortVectors whole vectors: four vectors a lane at most, or eight of a wave's.
constexpr int64_t kShortVectors = 512;
int lanes_of(int64_t vectors) { return vectors <= 32 ? 8 : (vectors <= 64 ? 16 : (vectors <= 128 ? 32 : 64)); }

// The backward's: at least 16 (65536 rows of 257: 19.1 us, with 8 lanes a row, whose stores are
// half as long, 24.9 us; the forward 10.3 us with 8 and 11.7 us with 16).
int grad_lanes_of(int64_t vectors) {
  if (vectors > kShortVectors) return kThreads;
  const int lanes = lanes_of(vectors);
  return lanes < 16 ? 16 : lanes;
}

// The workgroups of the backward a row: of a long row, with one vector more for a start between
// boundaries and one for the end.
int64_t grad_chunks(int64_t vectors) {
  return vectors <= kShortVectors ? 1 : (vectors + 2 + kGradVectors * kThreads - 1) / (kGradVectors * kThreads);
}

// Stretches a row is read in: one, but for a few rows of 65536 logits or more, whose exponentials are
// more work than one compute unit's share of the read (a row of 128000 bfloat16 by 1024 threads: 8.3 us;
// by 15 workgroups and a second launch that joins them: 5.3 us; 64 rows: 9.8 and 8.9 us; 128 rows: 10.4
// and 11.2 us; one row of 32000: 4.5 and 5.5 us; where both limits meet, 64 rows of 70000, 6.3 and 7.5 us).
int64_t stretches(int64_t rows, int64_t vocab) {
  if (rows > 64 || vocab < 65536) return 1;
  const int64_t want = 512 / (rows > 0 ? rows : 1), most = vocab / 8192;
  const int64_t n = want < most ? want : most;
  return n > 64 ? 64 : n;
}

int vector_of(int dtype) { return dtype == TI_F64 ? 2 : (dtype == TI_F32 ? 4 : 8); }

unsigned blocks_of(int64_t rows, int lanes) {
  const int64_t per = kThreads / lanes;
  return static_cast<unsigned>((rows + per - 1) / per);
}

}  // namespace

int64_t logprobs_rows(int64_t vocab, int dtype) {
  // (a launch holds less than 2^32 threads: the backward's are the most)
  const int64_t vectors = vocab / vector_of(dtype);
  return vocab > (int64_t{1} << 24) ? 0 : 0xFFFFFFFF / (grad_lanes_of(vectors) * grad_chunks(vectors)) - kThreads;
}

size_t logprobs_bytes(int64_t rows, int64_t vocab, int dtype) {
  const int64_t vectors = vocab / vector_of(dtype);
  if (vectors <= kShortVectors) return 0;
  const int64_t n = stretches(rows, vocab);
  return n < 2 ? 0 : static_cast<size_t>(rows * n) * (dtype == TI_F64 ? sizeof(Part<double, true>) : sizeof(Part<float, true>));
}

hipError_t logprobs(const LogprobArgs& a, void* work) {
  const Rows where{a.inner, a.outer_stride, a.row_stride};
  auto of = [&](auto zero, auto entropy) -> hipError_t {
    using T = decltype(zero);
    using A = typename AccOf<T>::type;
    constexpr bool ENT = decltype(entropy)::value;
    const auto* z = static_cast<const T*>(a.logits);
    const Results<A, ENT> out{static_cast<A*>(a.logp), static_cast<A*>(a.entropy), static_cast<A*>(a.stats), a.rows};
    const int vocab = static_cast<int>(a.vocab);
    const int64_t vectors = a.vocab / Vec<T>::kN;
    if (vectors <= kShortVectors) {
      const int lanes = lanes_of(vectors);
      auto go = [&](auto kernel) {
        kernel<<<dim3(blocks_of(a.rows, lanes)), dim3(kThreads), 0, a.stream>>>(z, a.targets, out, vocab, where, a.ignore, a.temperature);
      };
      if (lanes == 8) go(logprobs_short_kernel<T, ENT, 8, 4>);
      else if (lanes == 16) go(logprobs_short_kernel<T, ENT, 16, 4>);
      else if (lanes == 32) go(logprobs_short_kernel<T, ENT, 32, 4>);
      else if (vectors <= 256) go(logprobs_short_kernel<T, ENT, 64, 4>);
      else go(logprobs_short_kernel<T, ENT, 64, 8>);
      return hipGetLastError();
    }
    const int64_t n = stretches(a.rows, a.vocab);
    auto* parts = static_cast<Part<A, ENT>*>(n < 2 ? nullptr : work);
    auto go = [&](auto kernel, int threads) {
      kernel<<<dim3(static_cast<unsigned>(a.rows), static_cast<unsigned>(n)), dim3(threads), 0, a.stream>>>(
          z, a.targets, out, vocab, where, a.ignore, a.temperature, parts);
    };
    // (eight to sixteen vectors a thread, so that a row's start and its joining are little of its time and
    // a CU has several rows on the way; few rows by as many threads as there are. bfloat16: 8192 rows of
    // 128000 in 351, 343 and 330 us by 256, 512 and 1024 threads, 2048 of 50001 in 37.8, 36.6 and 40.4 us,
    // 8192 of 16000 in 50, 55 and 70 us; 16384 of 5000 by 64 threads 33 us, by 256 45 us)
    if (n > 1) go(logprobs_kernel<T, ENT, 256>, 256);
    else if (a.rows <= 512 || vectors > 12000) go(logprobs_kernel<T, ENT, 1024>, 1024);
    else if (vectors > 4096) go(logprobs_kernel<T, ENT, 512>, 512);
    else if (vectors > 1024) go(logprobs_kernel<T, ENT, 256>, 256);
    else go(logprobs_kernel<T, ENT, 64>, 64);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || n < 2) return e;
    logprobs_join_kernel<T, ENT><<<dim3(static_cast<unsigned>(a.rows)), dim3(64), 0, a.stream>>>(
        z, a.targets, out, vocab, where, a.ignore, a.temperature, parts, static_cast<int>(n));
    return hipGetLastError();
  };
  auto go = [&](auto zero) { return a.entropy != nullptr ? of(zero, std::true_type{}) : of(zero, std::false_type{}); };
  if (a.dtype == TI_F32) return go(float{});
  if (a.dtype == TI_F64) return go(double{});
  if (a.dtype == TI_BF16) return go(__bf16{});
  return go(_Float16{});
}

hipError_t logprobs_grad(const LogprobArgs& a, const void* g, const void* ge, void* grad) {
  const Rows where{a.inner, a.outer_stride, a.row_stride};
  auto of = [&](auto zero, auto entropy) {
    using T = decltype(zero);
    using A = typename AccOf<T>::type;
    constexpr bool ENT = decltype(entropy)::value;
    const int64_t vectors = a.vocab / Vec<T>::kN;
    const int lanes = grad_lanes_of(vectors);
    const int64_t chunks = grad_chunks(vectors);
    // (from both ends where the last-level cache, 256 MB, still has a good part of the logits, its rows read
    // beside those in memory: 524 MB forward and backward in 234 us and in turn 241 us; 2.1 GB in 1042 and
    // 1009 us; under 256 MB there is no difference)
    const double mb = static_cast<double>(a.rows) * static_cast<double>(a.vocab) * sizeof(T) / 1048576.0;
    const bool mixed = mb > 256.0 && mb <= 1024.0;
    auto go = [&](auto kernel) {
      kernel<<<dim3(static_cast<unsigned>(blocks_of(a.rows, lanes) * chunks)), dim3(kThreads), 0, a.stream>>>(
          static_cast<const T*>(a.logits), a.targets, static_cast<const A*>(a.stats), static_cast<const A*>(a.entropy),
          static_cast<const A*>(g), static_cast<const A*>(ge), static_cast<T*>(grad), a.rows, static_cast<int>(a.vocab),
          where, a.ignore, a.temperature, static_cast<unsigned>(chunks), mixed);
    };
    if (lanes == 16) go(logprobs_grad_kernel<T, ENT, 16>);
    else if (lanes == 32) go(logprobs_grad_kernel<T, ENT, 32>);
    else if (lanes == 64) go(logprobs_grad_kernel<T, ENT, 64>);
    else go(logprobs_grad_kernel<T, ENT, kThreads>);
    return hipGetLastError();
  };
  auto go = [&](auto zero) { return ge != nullptr ? of(zero, std::true_type{}) : of(zero, std::false_type{}); };
  if (a.dtype == TI_F32) return go(float{});
  if (a.dtype == TI_F64) return go(double{});
  if (a.dtype == TI_BF16) return go(__bf16{});
  return go(_Float16{});
}

}  // namespace ti
