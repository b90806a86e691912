// Losses over the log-probabilities of tokens, with their gradients: preference losses over pairs of
// sequences, and the clipped policy loss.
//
// The tokens of sequence i are those of the places [start(i), start(i + 1)) of the packed arrays, given
// by offsets or, for rows of one length, by i times that length; a masked token counts as absent,
// whatever its values. Sums run in float64; the policy loss's terms are of the tokens' type, and the first
// four of float32 are added in it.
//
// Preference: with x = l - l_ref, s_i the sum of x over the sequence's tokens (or their mean; 0 where
// there are none), the first half of the sequences chosen and the second half rejected, and
// h = s_chosen - s_rejected, a pair's loss is
//
//   logistic   -(1 - e) log sigmoid(b h) - e log sigmoid(-b h),   slope  b (e sigmoid(b h) - (1 - e) sigmoid(-b h))
//   hinge      max(0, 1 - b h),                                   slope  -b where b h < 1
//   squared    (h - 1 / (2 b))^2,                                 slope  2 (h - 1 / (2 b))
//
// and a token's gradient its pair's slope (over the sequence's tokens for a mean), negated in the
// rejected sequence.
//
// Policy: with r = exp(l - l_old), d = l_ref - l, a token's loss and gradient are
//
//   -min(r A, clip(r, lo, hi) A) + k (e^d - 1 - d),     -(r A where that is the smaller) - k (e^d - 1),
//
// times the token's weight: 1 / tokens, 1 / (sequences x the sequence's tokens), or 1.
#include <hip/hip_runtime.h>

#include <cmath>

#include "ti_common.h"
#include "ti_kernels.h"

namespace ti {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kPairThreads = 1024;
constexpr int64_t kPairBlocks = 512;

struct Sequences {
  const int64_t* offsets;  // null: rows of `len`
  int64_t count, len, total;
  // The start of sequence i (count: the end of the last), inside the arrays whatever the offsets are.
  __device__ __forceinline__ int64_t start(int64_t i) const {
    if (offsets == nullptr) return i * len;
    const int64_t v = offsets[i];
    return v < 0 ? 0 : (v > total ? total : v);
  }
  // Whether sequence i's offsets are what they have to be: from 0 to the total, not decreasing.
  __device__ __forceinline__ bool sound(int64_t i) const {
    if (offsets == nullptr) return true;
    const int64_t a = offsets[i], b = offsets[i + 1];
    return a <= b && a >= 0 && b <= total && (i > 0 || a == 0) && (i + 1 < count || b == total);
  }
  // The sequence that holds place j, of those from lo to below hi: the last that starts at or before j.
  __device__ __forceinline__ int64_t find(int64_t j, int64_t lo, int64_t hi) const {
    while (hi - lo > 1) {
      const int64_t mid = lo + (hi - lo) / 2;
      if (start(mid) <= j) lo = mid;
      else hi = mid;
    }
    return lo;
  }
};

// The sequences of a wave's places [begin, end) (begin < end), from lo to hi: one reading of 64 starts per factor
// of 64 of the sequences' number, and one more of the starts after lo.
struct Held {
  int64_t lo, hi;
  bool known;  // lane `skip` + k holds the start of lo + k, relative to begin, for all of them and the one after hi
  int skip, rel;
  __device__ __forceinline__ Held(const Sequences& seq, int64_t begin, int64_t end) {
    const int lane = threadIdx.x & 63;
    int64_t base, v;
    if (seq.offsets == nullptr) {
      base = wave_uniform(begin / seq.len);
      lo = base;
      v = base + lane <= seq.count ? seq.start(base + lane) : seq.total + 1;
    } else {
      int64_t from = 0, to = seq.count;
      while (true) {
        const int64_t step = (to - from + 63) >> 6, p = from + step * lane;
        v = p <= seq.count ? seq.start(p) : seq.total + 1;
        const int k = __popcll(__ballot(lane == 0 || (p < to && v <= begin))) - 1;
        if (step == 1) {
          base = from;
          lo = from + k;
          break;
        }
        from += step * k;
        to = from + step < to ? from + step : to;
      }
    }
    // (no sequence of these places from here on)
    const uint64_t past = __ballot(base + lane >= seq.count || v >= end);
    hi = past != 0 ? base + __builtin_ctzll(past) - 1 : seq.find(end - 1, lo, seq.count);
    known = past != 0;
    skip = static_cast<int>(lo - base);
    hi = wave_uniform(hi < lo ? lo : hi);  // (less: offsets that decrease)
    lo = wave_uniform(lo);
    const int64_t d = v - begin;
    rel = d < 0 ? 0 : (d > (1 << 30) ? 1 << 30 : static_cast<int>(d));
  }
};

// What the lanes of a wave wrote to shared memory is there for its other lanes (whose instructions keep their order).
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// The sequence, less held.lo, that starts at each of a wave's 256 U places from `begin` on, or -1, in its shared
// memory. (An empty sequence starts where another does, and has no place; the one at the first place goes without.)
template <int U>
__device__ __forceinline__ void starts_of(const Sequences& seq, const Held& held, int64_t begin, int* heads) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) heads[u * 256 + lane * 4 + i] = -1;
  wave_sync();
  if (held.known) {
    const int k = lane - held.skip, next = __shfl_down(held.rel, 1);
    if (k > 0 && k <= held.hi - held.lo && held.rel > 0 && held.rel < 256 * U && next > held.rel) heads[held.rel] = k;
  } else {
    for (int64_t i0 = held.lo; i0 <= held.hi; i0 += 64) {
      const int64_t i = i0 + lane;
      if (i <= held.hi) {
        const int64_t a = seq.start(i) - begin, b = seq.start(i + 1) - begin;
        if (a > 0 && a < 256 * U && b > a) heads[a] = static_cast<int>(i - held.lo);
      }
    }
  }
  wave_sync();
}

// The sequences, less held.lo, of the lane's four places whose starts these are, by the wave; open: the one before
// them, then the one after the wave's.
__device__ __forceinline__ void sequences_at(const int* heads, int& open, int (&at)[4]) {
  int id = -1;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int head = heads[i];
    id = head >= 0 ? head : id;
    at[i] = id;
  }
  const int lane = threadIdx.x & 63;
  const uint64_t with = __ballot(id >= 0), before = with & ((uint64_t{1} << lane) - 1);
  const int theirs = __shfl(id, before != 0 ? 63 - __builtin_clzll(before) : 0);
  const int base = before != 0 ? theirs : open;
#pragma unroll
  for (int i = 0; i < 4; ++i) at[i] = at[i] >= 0 ? at[i] : base;
  if (with != 0) open = __builtin_amdgcn_readlane(id, 63 - __builtin_clzll(with));
}

// The sum over the wave (all 64 lanes active), in every lane.
__device__ __forceinline__ double wave_sum(double v) { return wave_last_f64(wave_incl_f64(v)); }

// The same of whole numbers, whose sum is below 2^32: a scalar.
__device__ __forceinline__ uint32_t wave_total(uint32_t v) {
  v += dpp_i32<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v += dpp_i32<0x112, 0xF>(v);
  v += dpp_i32<0x114, 0xF>(v);
  v += dpp_i32<0x118, 0xF>(v);
  v += dpp_i32<0x142, 0xA>(v);  // row_bcast 15, 31
  v += dpp_i32<0x143, 0xC>(v);
  return __builtin_amdgcn_readlane(v, 63);
}

// The workgroup's sums of the values v, in every thread.
template <int NT, int K>
__device__ __forceinline__ void block_sums(double (&v)[K]) {
  __shared__ double part[K][NT / 64];
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = wave_sum(v[k]);
  __syncthreads();
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) part[k][threadIdx.x >> 6] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = 0.0;
#pragma unroll 4
    for (int w = 0; w < NT / 64; ++w) v[k] += part[k][w];
  }
}
template <int NT>
__device__ __forceinline__ double block_sum(double v) {
  double s[1] = {v};
  block_sums<NT>(s);
  return s[0];
}

// The same, and whether any thread's `any` was set, in every thread.
template <int NT>
__device__ __forceinline__ double block_sum(double v, bool& any) {
  __shared__ int flag[NT / 64];
  const bool wave = __any(any);
  if ((threadIdx.x & 63) == 0) flag[threadIdx.x >> 6] = wave;
  v = block_sum<NT>(v);  // (whose barriers come between)
  any = __any(flag[threadIdx.x % (NT / 64)]);
  return v;
}

// Four consecutive values of a token array at any alignment; those past the end zero.
template <typename T>
struct Four {
  T v[4];
  __device__ __forceinline__ void load_all(const T* __restrict__ p, int64_t j) { __builtin_memcpy(v, p + j, 4 * sizeof(T)); }
  __device__ __forceinline__ void load_some(const T* __restrict__ p, int64_t j, int64_t total) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = j + i < total ? p[j + i] : T(0);
  }
  __device__ __forceinline__ void load(const T* __restrict__ p, int64_t j, int64_t total) {
    if (j + 4 <= total)
      load_all(p, j);
    else
      load_some(p, j, total);
  }
  __device__ __forceinline__ void store(T* __restrict__ p, int64_t j, int64_t total) const {
    if (j + 4 <= total) {
      // (past the caches: 16384 x 1024 tokens' policy loss 64.1 -> 59.8 us; such loads made it 67.3 us)
      using Values = T __attribute__((ext_vector_type(4), aligned(sizeof(T))));
      __builtin_nontemporal_store(Values{v[0], v[1], v[2], v[3]}, reinterpret_cast<Values*>(p + j));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (j + i < total) p[j + i] = v[i];
    }
  }
};

// --- preference --------------------------------------------------------------------------------

struct Sum {
  double s, n;
};

// Inclusive sums over the lanes, each from the lane `from` on (all 64 lanes active): within rows of 16, then the row
// before (15, 47) and the half before (31).
__device__ __forceinline__ void scan_from(double& s, int& n, int lane, int from) {
  auto add = [&](double ds, int dn, bool in) {
    s += in ? ds : 0.0;
    n += in ? dn : 0;
  };
  add(dpp_f64<0x111, 0xF>(s), dpp_i32<0x111, 0xF>(n), lane - from >= 1);
  add(dpp_f64<0x112, 0xF>(s), dpp_i32<0x112, 0xF>(n), lane - from >= 2);
  add(dpp_f64<0x114, 0xF>(s), dpp_i32<0x114, 0xF>(n), lane - from >= 4);
  add(dpp_f64<0x118, 0xF>(s), dpp_i32<0x118, 0xF>(n), lane - from >= 8);
  add(dpp_f64<0x142, 0xA>(s), dpp_i32<0x142, 0xA>(n), from < (lane & 48));
  add(dpp_f64<0x143, 0xC>(s), dpp_i32<0x143, 0xC>(n), from < 32);
}

// The sums of every sequence, a wave a tile of 256 U places, four a lane at a time. A sequence's part in
// a tile goes to
//
//   first[tile]   if it holds the tile's first place,
//   last[tile]    else, if it goes on to the tile's end (of a whole tile),
//   whole[i]      else: it begins and ends inside,
//
// so that every value has one writer, and a sequence's sum is its first part and the `first` parts of
// the tiles that follow. A tile of several sequences is summed by a segmented scan over the lanes: `heads`,
// the wave's shared memory, holds the sequence that starts at each of its places.
//
// Bound by its reads where sequences are long (2048 sequences of 1 to 8191 tokens, 75 MB: 18.1 us, 4.1 TB/s;
// read four bytes a lane, 64 places at a time, 46 us), by the scan's instructions where they are short.
template <typename T, int U>
__device__ __forceinline__ void tile_sums(const T* __restrict__ logps, const T* __restrict__ ref,
                                          const uint8_t* __restrict__ mask, const Sequences& seq, int64_t tile, int* heads,
                                          Sum* __restrict__ first, Sum* __restrict__ last, Sum* __restrict__ whole) {
  constexpr int kPlaces = 256 * U;
  const int lane = threadIdx.x & 63;
  const int64_t begin = tile * kPlaces;
  if (begin >= seq.total) return;
  const int size = seq.total - begin < kPlaces ? static_cast<int>(seq.total - begin) : kPlaces;
  Four<T> x[U], y[U];
  Four<uint8_t> m[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t j = begin + u * 256 + lane * 4;
    x[u].load(logps, j, seq.total);
    if (ref != nullptr) y[u].load(ref, j, seq.total);
    else y[u] = Four<T>{};
    if (mask != nullptr) m[u].load(mask, j, seq.total);
    else m[u] = Four<uint8_t>{{j < seq.total, j + 1 < seq.total, j + 2 < seq.total, j + 3 < seq.total}};
  }
  const Held held(seq, begin, begin + size);
  if (held.lo == held.hi) {
    double v = 0.0;
    int count = 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool kept = m[u].v[i] != 0;
        v += kept ? static_cast<double>(x[u].v[i]) - static_cast<double>(y[u].v[i]) : 0.0;
        count += __popcll(__ballot(kept));
      }
    v = wave_sum(v);
    if (lane == 0) first[tile] = Sum{v, static_cast<double>(count)};
    return;
  }
  starts_of<U>(seq, held, begin, heads);
  double open_s = 0.0;  // the open sequence's sum and count so far, and which it is
  int open_n = 0, open = 0;
  bool is_first = true;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    // the lane's four places: of the sequence that is open before them (left), of those that begin and end in
    // them, of the one that is open after them (s, n)
    double s = 0.0, left = 0.0;
    int n = 0, left_n = 0, mine = -1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int head = heads[u * 256 + lane * 4 + i];
      if (head >= 0) {
        if (mine >= 0) {
          whole[held.lo + mine] = Sum{s, static_cast<double>(n)};
        } else {
          left = s;
          left_n = n;
        }
        mine = head;
        s = 0.0;
        n = 0;
      }
      const bool kept = m[u].v[i] != 0;
      s += kept ? static_cast<double>(x[u].v[i]) - static_cast<double>(y[u].v[i]) : 0.0;
      n += kept ? 1 : 0;
    }
    const uint64_t with = __ballot(mine >= 0), before = with & ((uint64_t{1} << lane) - 1);
    const uint64_t upto = mine >= 0 ? before | (uint64_t{1} << lane) : before;
    // sums from the lane that last held a start on
    const int from = upto != 0 ? 63 - __builtin_clzll(upto) : 0;
    scan_from(s, n, lane, from);
    if (upto == 0) {
      s += open_s;
      n += open_n;
    }
    double s1 = __shfl_up(s, 1);
    int n1 = __shfl_up(n, 1);
    if (lane == 0) {
      s1 = open_s;
      n1 = open_n;
    }
    const int past = before != 0 ? 63 - __builtin_clzll(before) : 0;
    const int theirs = __shfl(mine, past);
    if (mine >= 0)
      (before == 0 && is_first ? first[tile] : whole[held.lo + (before == 0 ? open : theirs)]) =
          Sum{s1 + left, static_cast<double>(n1 + left_n)};
    open_s = __shfl(s, 63);
    open_n = __shfl(n, 63);
    if (with != 0) {
      is_first = false;
      open = __shfl(mine, 63 - __builtin_clzll(with));
    }
  }
  if (lane == 0)
    (is_first ? first[tile] : (size == kPlaces ? last[tile] : whole[held.lo + open])) = Sum{open_s, static_cast<double>(open_n)};
}

// The sum over the G lanes of a group of the wave (all 64 lanes active), in the group's last lane.
template <int G>
__device__ __forceinline__ double group_sum(double v) {
  static_assert(G == 4 || G == 32);
  v += dpp_f64<0x111, 0xF>(v);
  v += dpp_f64<0x112, 0xF>(v);
  if constexpr (G == 4) return v;
  v += dpp_f64<0x114, 0xF>(v);
  v += dpp_f64<0x118, 0xF>(v);
  v += dpp_f64<0x142, 0xA>(v);
  return v;
}

// The sum of sequence i, by G lanes, in the last of them; NaN of -1 where its offsets are not sound.
template <int G>
__device__ __forceinline__ Sum sum_of(const Sequences& seq, int64_t i, int tile_places, const Sum* __restrict__ first,
                                      const Sum* __restrict__ last, const Sum* __restrict__ whole) {
  const int lane = threadIdx.x % G;
  const int64_t a = seq.start(i), b = seq.start(i + 1);
  Sum v{0.0, 0.0};
  if (a < b) {
    const int64_t t0 = a / tile_places, t1 = (b - 1) / tile_places;
    if (lane == 0) v = a == t0 * tile_places ? first[t0] : (b < (t0 + 1) * tile_places ? whole[i] : last[t0]);
    // (eight on their way at a time, which the compiler's own schedule does not keep: two sequences of 8 million
    // tokens in 52.7 us, one after another 162 us)
    constexpr int kAhead = 8;
    int64_t t = t0 + 1 + lane;
    for (; t + (kAhead - 1) * G <= t1; t += kAhead * G) {
      Sum w[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) w[i] = first[t + i * G];
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        v.s += w[i].s;
        v.n += w[i].n;
      }
    }
    for (; t <= t1; t += G) {
      const Sum w = first[t];
      v.s += w.s;
      v.n += w.n;
    }
  }
  v.s = group_sum<G>(v.s);
  v.n = group_sum<G>(v.n);
  if (!seq.sound(i)) v = Sum{quiet_nan<double>(), -1.0};
  return v;
}

struct Pair {
  double loss, slope;
};

__device__ __forceinline__ Pair pair_loss(double h, int kind, double beta, double smoothing) {
  if (kind == TI_LOSS_HINGE) {
    const double v = 1.0 - beta * h;
    return {v < 0.0 ? 0.0 : v, v > 0.0 ? -beta : (v <= 0.0 ? 0.0 : v)};
  }
  if (kind == TI_LOSS_SQUARED) {
    const double v = h - 0.5 / beta;
    return {v * v, 2.0 * v};
  }
  const double x = beta * h, e = exp(-fabs(x));
  const double soft = log1p(e);
  const double up = x > 0.0 ? x : 0.0, down = x < 0.0 ? -x : 0.0;
  const double small = e / (1.0 + e), large = 1.0 / (1.0 + e);  // sigmoid(-|x|), sigmoid(|x|)
  const double plus = x > 0.0 ? large : small, minus = x > 0.0 ? small : large;
  // (no product of an infinite part with a smoothing of zero)
  return {(1.0 - smoothing) * (soft + down) + (smoothing > 0.0 ? smoothing * (soft + up) : 0.0),
          beta * (smoothing * plus - (1.0 - smoothing) * minus)};
}

template <typename T, int U>
__global__ __launch_bounds__(kThreads) void preference_sums_kernel(const T* __restrict__ logps, const T* __restrict__ ref,
                                                                   const uint8_t* __restrict__ mask, Sequences seq,
                                                                   Sum* __restrict__ first, Sum* __restrict__ last,
                                                                   Sum* __restrict__ whole) {
  __shared__ __attribute__((aligned(16))) int heads[kWaves][256 * U];
  const int wave = threadIdx.x >> 6;
  tile_sums<T, U>(logps, ref, mask, seq, static_cast<int64_t>(blockIdx.x) * kWaves + wave, heads[wave], first, last, whole);
}

template <typename T>
struct PairArgs {
  int kind, average, reduction;
  double beta, smoothing;
  T *loss, *chosen, *rejected, *slopes;
  // What a pair's loss is times in the reduced one.
  __device__ __forceinline__ double scale(int64_t pairs) const {
    return reduction == TI_REDUCE_MEAN ? 1.0 / static_cast<double>(pairs) : 1.0;
  }
};

// Bound by latency: a chain of three reads (a sequence's starts, its parts, its pair's other half) and the
// scalar formula (1024 pairs, one a wave: 6.9 us). Sequences of less than a tile take four lanes each, so
// that a wave has eight pairs on the way (200000 pairs of short sequences: the forward 226 us with 32 lanes each,
// 89 us with four).
//
// The pairs from `begin` on, G lanes a sequence and 2 G a pair (the chosen sequence by the first half, the
// rejected one by the second), `step` pairs apart: their results, and the sum of their losses in this
// workgroup, and whether it met offsets that are not sound.
template <int NT, int G, typename T>
__device__ __forceinline__ double pair_losses(const Sequences& seq, int64_t begin, int64_t step, int tile_places,
                                              const Sum* __restrict__ first, const Sum* __restrict__ last,
                                              const Sum* __restrict__ whole, const PairArgs<T>& a, bool& bad) {
  const int64_t pairs = seq.count / 2;
  const int lane = threadIdx.x & 63, side = (lane / G) & 1;
  const double scale = a.scale(pairs);
  double all = 0.0;
  for (int64_t p0 = begin; p0 < pairs; p0 += step) {  // (the same turns for every lane of a wave)
    const int64_t p = p0 + lane / (2 * G);
    const bool in = p < pairs;
    const Sum mine = sum_of<G>(seq, in ? (side != 0 ? pairs + p : p) : 0, tile_places, first, last, whole);
    const int at = lane / (2 * G) * (2 * G) + G - 1;  // (the chosen one's last lane; the rejected one's G on)
    const Sum c{__shfl(mine.s, at), __shfl(mine.n, at)}, j{__shfl(mine.s, at + G), __shfl(mine.n, at + G)};
    if (!in || lane % (2 * G) != 0) continue;
    bad = bad || c.n < 0.0 || j.n < 0.0;
    const double wc = a.average && c.n > 0.0 ? 1.0 / c.n : 1.0, wj = a.average && j.n > 0.0 ? 1.0 / j.n : 1.0;
    const double sc = c.s * wc, sj = j.s * wj;
    const Pair v = pair_loss(sc - sj, a.kind, a.beta, a.smoothing);
    a.chosen[p] = static_cast<T>(a.beta * sc);
    a.rejected[p] = static_cast<T>(a.beta * sj);
    if (a.slopes != nullptr) {
      a.slopes[p] = static_cast<T>(v.slope * wc * scale);
      a.slopes[pairs + p] = static_cast<T>(-v.slope * wj * scale);
    }
    if (a.reduction == TI_REDUCE_NONE) a.loss[p] = static_cast<T>(v.loss);
    all += v.loss;
  }
  return a.reduction == TI_REDUCE_NONE ? 0.0 : block_sum<NT>(all, bad);
}

// Offsets that are not sound leave no token with a gradient to go by: every slope NaN, by one workgroup, all of
// whose threads have the same `bad`.
template <int NT, typename T>
__device__ __forceinline__ void void_slopes(bool bad, T* __restrict__ slopes, int64_t count) {
  if (!bad || slopes == nullptr) return;
  for (int64_t i = threadIdx.x; i < count; i += NT) slopes[i] = quiet_nan<T>();
}

// A workgroup's sum of its pairs' losses, and whether it met offsets that are not sound.
struct PairPart {
  double all;
  int64_t bad;
};

template <typename T, int G>
__global__ __launch_bounds__(kPairThreads) void preference_pairs_kernel(Sequences seq, int tile_places,
                                                                        const Sum* __restrict__ first,
                                                                        const Sum* __restrict__ last,
                                                                        const Sum* __restrict__ whole, PairArgs<T> a,
                                                                        PairPart* __restrict__ parts) {
  constexpr int kEach = 32 / G;  // pairs a wave
  const int64_t wave = static_cast<int64_t>(blockIdx.x) * (kPairThreads / 64) + (threadIdx.x >> 6);
  bool bad = false;
  const double all = pair_losses<kPairThreads, G>(seq, wave * kEach, static_cast<int64_t>(gridDim.x) * (kPairThreads / 64) * kEach,
                                                  tile_places, first, last, whole, a, bad);
  if (a.reduction == TI_REDUCE_NONE) return;
  if (gridDim.x == 1) void_slopes<kPairThreads>(bad, a.slopes, seq.count);
  if (threadIdx.x != 0) return;
  if (gridDim.x == 1) a.loss[0] = static_cast<T>(all * a.scale(seq.count / 2));
  else parts[blockIdx.x] = PairPart{all, bad};
}

// Few tokens in one workgroup: their sums, then the pairs. (Four pairs, 2620 tokens: 6.5 us, in two
// launches 8.5 us.)
template <typename T>
__global__ __launch_bounds__(kPairThreads) void preference_small_kernel(const T* __restrict__ logps,
                                                                        const T* __restrict__ ref,
                                                                        const uint8_t* __restrict__ mask, Sequences seq,
                                                                        Sum* first, Sum* last, Sum* whole, PairArgs<T> a) {
  constexpr int kEach = kPairThreads / 64;
  __shared__ __attribute__((aligned(16))) int heads[kEach][256];
  for (int64_t tile = threadIdx.x >> 6; tile * 256 < seq.total; tile += kEach)
    tile_sums<T, 1>(logps, ref, mask, seq, tile, heads[threadIdx.x >> 6], first, last, whole);
  __syncthreads();
  bool bad = false;
  const double all = pair_losses<kPairThreads, 32>(seq, threadIdx.x >> 6, kEach, 256, first, last, whole, a, bad);
  if (a.reduction == TI_REDUCE_NONE) return;
  void_slopes<kPairThreads>(bad, a.slopes, seq.count);
  if (threadIdx.x == 0) a.loss[0] = static_cast<T>(all * a.scale(seq.count / 2));
}

template <typename T>
__global__ __launch_bounds__(kPairThreads) void preference_mean_kernel(const PairPart* __restrict__ parts, int count,
                                                                       double scale, T* __restrict__ loss,
                                                                       T* __restrict__ slopes, int64_t sequences) {
  double all = 0.0;
  bool bad = false;
  for (int i = threadIdx.x; i < count; i += kPairThreads) {
    const PairPart part = parts[i];
    all += part.all;
    bad = bad || part.bad != 0;
  }
  all = block_sum<kPairThreads>(all, bad);
  void_slopes<kPairThreads>(bad, slopes, sequences);
  if (threadIdx.x == 0) loss[0] = static_cast<T>(all * scale);
}

// Each token's gradient, its sequence's slope times the upstream one. Bound by its stores (16384 sequences of
// 1024, 84 MB: 13.1 us, 6.4 TB/s) and, where tiles hold several sequences, by the latency of finding them
// (8.4M tokens of 1 to 8191 each, 42 MB: 11.4 us, 3.7 TB/s; the mask read after the search 11.8 us).
template <typename T, int U>
__global__ __launch_bounds__(kThreads) void preference_grad_kernel(const uint8_t* __restrict__ mask, Sequences seq,
                                                                   const T* __restrict__ slopes,
                                                                   const T* __restrict__ g, int per_pair,
                                                                   T* __restrict__ grad) {
  const int64_t pairs = seq.count / 2;
  const int lane = threadIdx.x & 63;
  const int64_t begin = (static_cast<int64_t>(blockIdx.x) * kWaves + (threadIdx.x >> 6)) * (256 * U);
  if (begin >= seq.total) return;
  const int64_t end = begin + 256 * U < seq.total ? begin + 256 * U : seq.total;
  Four<uint8_t> m[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (mask != nullptr) m[u].load(mask, begin + u * 256 + lane * 4, seq.total);
    else m[u] = Four<uint8_t>{{1, 1, 1, 1}};
  }
  const Held held(seq, begin, end);
  auto of = [&](int64_t at) { return slopes[at] * g[per_pair ? (at < pairs ? at : at - pairs) : 0]; };
  const bool one = held.lo == held.hi;
  const T all = one ? of(held.lo) : T(0);
  __shared__ __attribute__((aligned(16))) int starts[kWaves][256 * U];
  int* heads = starts[threadIdx.x >> 6];
  if (!one) starts_of<U>(seq, held, begin, heads);
  int open = 0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int t = u * 256 + lane * 4;
    int at[4];
    if (!one) sequences_at(heads + t, open, at);
    Four<T> d;
#pragma unroll
    for (int i = 0; i < 4; ++i) d.v[i] = m[u].v[i] != 0 ? (one ? all : of(held.lo + at[i])) : T(0);
    d.store(grad, begin + t, seq.total);
  }
}

// --- policy ------------------------------------------------------------------------------------

// e^x. In float32 2^t of the rounded t = x log2(e), times 1 + lo ln(2) for what t lost, (lo: t's rounding
// and that of the constant); past |t| = 128 the power alone, which is 0 or infinite there. What is below
// 2^-126 is 0.
__device__ __forceinline__ float exp_of(float x) {
  constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
  constexpr float kRest = static_cast<float>(1.44269504088896340736 - static_cast<double>(kLog2e));
  const float t = x * kLog2e, lo = __builtin_fmaf(x, kRest, __builtin_fmaf(x, kLog2e, -t));
  const float e = __builtin_amdgcn_exp2f(t);
  return __builtin_fabsf(t) < 128.0f ? __builtin_fmaf(e, lo * kLn2, e) : e;
}
__device__ __forceinline__ double exp_of(double x) { return exp(x); }

// up = e^d - 1 and rest = e^d - 1 - d of four d, to a few roundings of their own values: the power series
// where they would cancel (|d| <= 1/2: terms to d^9 / 9! for float, the rest below 2^-30 of the first; to
// d^17 / 17! for double), and the exponential where a d is past that.
template <typename T>
__device__ __forceinline__ void exp_rest(const T (&d)[4], T (&up)[4], T (&rest)[4]) {
  // sum over k = 2..kTerms of d^(k - 2) / k!, from the last term
  constexpr int kTerms = sizeof(T) == 4 ? 9 : 17;
  constexpr auto over_factorial = [](int k) {
    double f = 1.0;
    for (int i = 2; i <= k; ++i) f *= i;
    return static_cast<T>(1.0 / f);
  };
  bool near = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    T t = over_factorial(kTerms);
#pragma unroll
    for (int k = kTerms - 1; k >= 2; --k) t = t * d[i] + over_factorial(k);
    rest[i] = t * d[i] * d[i];
    up[i] = d[i] + rest[i];
    near = near && d[i] >= T(-0.5) && d[i] <= T(0.5);
  }
  if (near) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const T e = exp_of(d[i]);
    if (!(d[i] >= T(-0.5) && d[i] <= T(0.5))) {
      up[i] = e - T(1);
      rest[i] = e == T(INFINITY) ? e : up[i] - d[i];
    }
  }
}

// The clip's bounds, and what they lost when they were rounded: a float32 bound of 1.2 moves every clipped
// token the same way (8e-7 of the loss of 16384 samples of 1024 tokens, whose advantages nearly cancel), so
// the sums get it back.
template <typename T>
struct Clip {
  T low, high, low_lost, high_lost;
  Clip(double lo, double hi)
      : low(static_cast<T>(lo)), high(static_cast<T>(hi)),
        low_lost(static_cast<T>(lo - static_cast<double>(low))), high_lost(static_cast<T>(hi - static_cast<double>(high))) {}
};

// Four tokens' losses and their derivatives.
template <typename T>
struct Tokens {
  T loss[4], more[4], kl[4], grad[4];  // the loss is loss + more
  bool cut[4];
  __device__ __forceinline__ Tokens(const T (&l)[4], const T (&old)[4], const T (&a)[4], const Clip<T>& clip) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T r = exp_of(l[i] - old[i]);
      const bool under = r < clip.low;
      const T free = r * a[i], kept = (under ? clip.low : (r > clip.high ? clip.high : r)) * a[i];
      cut[i] = kept < free;
      loss[i] = -(cut[i] ? kept : free);
      more[i] = cut[i] ? -((under ? clip.low_lost : clip.high_lost) * a[i]) : T(0);
      grad[i] = cut[i] ? T(0) : -free;
      kl[i] = T(0);
    }
  }
  __device__ __forceinline__ void diverge(const T (&l)[4], const T (&ref)[4], T k) {
    T d[4], up[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = ref[i] - l[i];
    exp_rest(d, up, kl);
    if (k == T(0)) return;  // (no product of an infinite divergence with a coefficient of zero)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      loss[i] += k * kl[i];
      grad[i] -= k * up[i];
    }
  }
};

// 1 / x of a finite x >= 1, to a rounding or two: the hardware's approximation and two steps of Newton's method
// (the division takes twice the instructions and registers).
__device__ __forceinline__ double reciprocal(double x) {
  double r = __builtin_amdgcn_rcp(x);
  r = __builtin_fma(__builtin_fma(-x, r, 1.0), r, r);
  return __builtin_fma(__builtin_fma(-x, r, 1.0), r, r);
}

// A workgroup's sums; n: its tokens, or NaN where an offset is not what it has to be.
struct PolicySums {
  double loss, kl, cut, n;
};

constexpr int kCountThreads = 1024;
constexpr int kCountBlocks = 256, kWeightBlocks = 4096;

// The nonzero bytes of p[a, b) of p[0, total), by `lanes` threads, this one's share.
__device__ __forceinline__ int64_t nonzero(const uint8_t* __restrict__ p, int64_t a, int64_t b, int64_t total, int lane,
                                           int lanes) {
  int64_t n = 0;
  int64_t j = a + static_cast<int64_t>(lane) * 16;
  // (0x80 in each byte that is not zero)
  auto marks = [](uint32_t w) { return (((w & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) | w) & 0x80808080u; };
#pragma unroll 4
  for (; j + 16 <= b; j += static_cast<int64_t>(lanes) * 16) {
    uint32_t w[4];
    __builtin_memcpy(w, p + j, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) n += __popc(marks(w[i]));
  }
  if (j >= b) return n;
  const int rest = static_cast<int>(b - j);
  if (j + 16 <= total) {  // (past b, but inside the array)
    uint32_t w[4];
    __builtin_memcpy(w, p + j, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = rest - 4 * i;
      n += k > 0 ? __popc(marks(w[i]) & (k < 4 ? (1u << (8 * k)) - 1 : ~0u)) : 0;
    }
  } else {
    for (int i = 0; i < rest; ++i) n += p[j + i] != 0 ? 1 : 0;
  }
  return n;
}

// What a mask says of the tokens' weights, by one workgroup of `blocks` of kCountThreads: for
// TI_REDUCE_SEQUENCES the weight of each sequence's tokens, counted by LANES threads a sequence; else the
// tokens of this workgroup's share of the places (the result).
template <int LANES>
__device__ __forceinline__ double count_tokens(const uint8_t* __restrict__ mask, const Sequences& seq, int reduction,
                                               int block, int blocks, double* __restrict__ weights) {
  const int64_t threads = static_cast<int64_t>(blocks) * kCountThreads;
  if (reduction != TI_REDUCE_SEQUENCES) {
    const int t = block * kCountThreads + static_cast<int>(threadIdx.x);
    return block_sum<kCountThreads>(static_cast<double>(nonzero(mask, 0, seq.total, seq.total, t, static_cast<int>(threads))));
  }
  const double share = 1.0 / static_cast<double>(seq.count);
  const int lane = threadIdx.x % LANES;
  // (every group of a workgroup takes as many turns: they meet in the sums)
  for (int64_t i0 = static_cast<int64_t>(block) * (kCountThreads / LANES); i0 < seq.count; i0 += threads / LANES) {
    const int64_t i = i0 + threadIdx.x / LANES;
    double k = i < seq.count ? static_cast<double>(nonzero(mask, seq.start(i), seq.start(i + 1), seq.total, lane, LANES)) : 0.0;
    if constexpr (LANES == kCountThreads) {
      k = block_sum<kCountThreads>(k);
    } else if constexpr (LANES == 64) {
      k = wave_sum(k);
    } else {
#pragma unroll
      for (int d = LANES / 2; d > 0; d >>= 1) k += __shfl_xor(k, d);
    }
    if (lane == 0 && i < seq.count) weights[i] = share / (k > 0.0 ? k : 1.0);
  }
  return 0.0;
}

// One read of the mask, 16 bytes a thread (16.8 MB: 5.4 us), where a mean's weights depend on it. It comes
// first, so that the pass over the tokens can write gradients with their weights: one that left them to be
// weighted by the backward took 102 us a call for 16384 x 1024 tokens, forward and backward, where this took 77 us.
template <int LANES>
__global__ __launch_bounds__(kCountThreads) void policy_count_kernel(const uint8_t* __restrict__ mask, Sequences seq,
                                                                     int reduction, uint32_t* __restrict__ tokens,
                                                                     double* __restrict__ weights) {
  const double n = count_tokens<LANES>(mask, seq, reduction, blockIdx.x, gridDim.x, weights);
  if (threadIdx.x == 0 && reduction != TI_REDUCE_SEQUENCES) tokens[blockIdx.x] = static_cast<uint32_t>(n);
}

// The counts of `blocks` workgroups (a multiple of four, at most kCountBlocks), four a lane, and their sum, or 1 of
// nothing, by the wave: in whole numbers of 16 bits and the rest, whose sums over the lanes need one instruction a step.
struct Counts {
  uint32_t k[4] = {0, 0, 0, 0};
  __device__ __forceinline__ void load(const uint32_t* __restrict__ counts, int blocks) {
    static_assert(kCountBlocks <= 256);
    const int i = (threadIdx.x & 63) * 4;
    if (i < blocks) __builtin_memcpy(k, counts + i, 16);
  }
  __device__ __forceinline__ double sum() const {
    const uint32_t own = k[0] + k[1] + k[2] + k[3];
    const uint32_t low = wave_total(own & 0xFFFFu), high = wave_total(own >> 16);
    const double n = static_cast<double>(high) * 65536.0 + static_cast<double>(low);
    return n >= 1.0 ? n : 1.0;
  }
};

// Whether an offset among this thread's share of them is not what it has to be.
__device__ __forceinline__ bool unsound(const Sequences& seq, int64_t thread, int64_t threads) {
  bool bad = false;
  if (seq.offsets != nullptr)
    for (int64_t i = thread; i < seq.count; i += threads) bad = bad || !seq.sound(i);
  return bad;
}

template <typename T>
struct PolicyInputs {
  const T *logps, *old, *adv, *ref;
  const uint8_t* mask;
  int adv_each, reduction;
  Clip<T> clip;
  T kl_coef;
  T* grad;
};

struct PolicyPart {
  double sums[2] = {0.0, 0.0};  // this lane's loss and divergence
  int cut = 0, n = 0;           // the wave's
};

// The tokens of the wave's 256 U places from `begin` on: their gradients written, their sums in v. weight: a
// token's where it is the same for all (with `tokens`: that of their sum); for TI_REDUCE_SEQUENCES they are in
// `weights`, by the sequence, or (null) its length's.
template <typename T, int U>
__device__ __forceinline__ void policy_places(const PolicyInputs<T>& in, const Sequences& seq, int64_t begin, int* heads, double weight,
                                              const uint32_t* __restrict__ tokens, int count_blocks, const double* weights,
                                              PolicyPart& v) {
  if (begin >= seq.total) return;
  const int lane = threadIdx.x & 63;
  const int64_t end = begin + 256 * U < seq.total ? begin + 256 * U : seq.total;
  Four<T> l, o, a, r;
  Four<uint8_t> m{{1, 1, 1, 1}};
  auto load = [&](int64_t j) {
    if (j + 4 <= seq.total) {
      l.load_all(in.logps, j);
      o.load_all(in.old, j);
      if (in.ref != nullptr) r.load_all(in.ref, j);
      if (in.adv_each) a.load_all(in.adv, j);
      if (in.mask != nullptr) m.load_all(in.mask, j);
    } else {
      l.load_some(in.logps, j, seq.total);
      o.load_some(in.old, j, seq.total);
      if (in.ref != nullptr) r.load_some(in.ref, j, seq.total);
      if (in.adv_each) a.load_some(in.adv, j, seq.total);
      if (in.mask != nullptr) m.load_some(in.mask, j, seq.total);
    }
  };
  Counts counts;
  if (tokens != nullptr) counts.load(tokens, count_blocks);
  load(begin + lane * 4);  // (on its way while the wave's sequences are looked for)
  const bool by_sequence = in.reduction == TI_REDUCE_SEQUENCES, sequences = by_sequence || !in.adv_each;
  const Held held(sequences ? seq : Sequences{nullptr, 1, seq.total, seq.total}, begin, end);
  const bool one = held.lo == held.hi;
  if (tokens != nullptr) weight = reciprocal(counts.sum());  // (the mean's weight by the mask)
  // what a sequence says of its tokens, a lane each where they are few
  auto weight_of = [&](int64_t i) {
    if (weights != nullptr) return weights[i];
    const int64_t size = seq.start(i + 1) - seq.start(i);
    return reciprocal(static_cast<double>(seq.count) * static_cast<double>(size > 0 ? size : 1));
  };
  const bool few = held.hi - held.lo < 64;
  const int64_t mine = held.lo + lane < held.hi ? held.lo + lane : held.hi;
  const T adv = in.adv_each ? T(0) : in.adv[mine];
  const double own = by_sequence ? weight_of(mine) : 0.0;
  if (one && by_sequence) weight = own;
  weight = __builtin_bit_cast(double, wave_uniform(__builtin_bit_cast(int64_t, weight)));  // (a scalar register's)
  const T each = static_cast<T>(weight);
  if (!one) starts_of<U>(seq, held, begin, heads);
  int open = 0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int t = u * 256 + lane * 4;
    int at[4];
    if (u > 0) load(begin + t);
    if (!one) sequences_at(heads + t, open, at);
    if (!in.adv_each) {
#pragma unroll
      for (int i = 0; i < 4; ++i) a.v[i] = one ? adv : (few ? __shfl(adv, at[i]) : in.adv[held.lo + at[i]]);
    }
    // (all four computed, whatever the mask; four tokens' sums are float32, in float64 from there on)
    Tokens<T> x(l.v, o.v, a.v, in.clip);
    if (in.ref != nullptr) x.diverge(l.v, r.v, in.kl_coef);
    bool kept[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) kept[i] = m.v[i] != 0 && (in.mask != nullptr || begin + t + i < seq.total);
    Four<T> d;
    T kl = T(0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      d.v[i] = kept[i] ? x.grad[i] : T(0);
      kl += kept[i] ? x.kl[i] : T(0);
      v.cut += __popcll(__ballot(kept[i] && x.cut[i]));
      v.n += __popcll(__ballot(kept[i]));
    }
    if (by_sequence && !one) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!few) __builtin_amdgcn_sched_barrier(0);  // (one after another: registers)
        const double w = few ? __shfl(own, at[i]) : weight_of(held.lo + at[i]);
        v.sums[0] += kept[i] ? (static_cast<double>(x.loss[i]) + static_cast<double>(x.more[i])) * w : 0.0;
        d.v[i] *= static_cast<T>(w);
      }
    } else {
      T loss = T(0), more = T(0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        loss += kept[i] ? x.loss[i] : T(0);
        more += kept[i] ? x.more[i] : T(0);
        d.v[i] *= each;
      }
      v.sums[0] += (static_cast<double>(loss) + static_cast<double>(more)) * weight;
    }
    v.sums[1] += static_cast<double>(kl);
    if (in.grad != nullptr) d.store(in.grad, begin + t, seq.total);
  }
}

// The workgroup's sums, in thread 0 (all other threads': no matter); bad: whether this thread saw an unsound offset.
// (By way of shared memory: a sum over the lanes of each wave would take as many instructions as a token's loss.)
template <int NT>
__device__ __forceinline__ PolicySums policy_sums(const PolicyPart& v, bool bad) {
  __shared__ double part[2][NT];
  __shared__ int cut[NT / 64], n[NT / 64];
  const bool any = __any(bad);
#pragma unroll
  for (int k = 0; k < 2; ++k) part[k][threadIdx.x] = v.sums[k];
  if ((threadIdx.x & 63) == 0) {
    cut[threadIdx.x >> 6] = v.cut;
    n[threadIdx.x >> 6] = any ? -1 : v.n;
  }
  __syncthreads();
  PolicySums all{0.0, 0.0, 0.0, 0.0};
  if (threadIdx.x >= 64) return all;
#pragma unroll 4
  for (int w = 0; w < NT / 64; ++w) {
    all.loss += part[0][w * 64 + threadIdx.x];
    all.kl += part[1][w * 64 + threadIdx.x];
    all.cut += cut[w];
    all.n += n[w] < 0 ? quiet_nan<double>() : n[w];
  }
  all.loss = wave_sum(all.loss);
  all.kl = wave_sum(all.kl);
  return all;
}

// Offsets that are not sound leave no token with a gradient to go by: that of every unmasked one NaN, by one
// workgroup. (Written once the pass that wrote gradients is over, so that it costs the others nothing.)
template <int NT, typename T>
__device__ __forceinline__ void void_gradient(const uint8_t* __restrict__ mask, int64_t total, T* __restrict__ grad) {
  if (grad == nullptr) return;
#pragma unroll 4
  for (int64_t j = static_cast<int64_t>(threadIdx.x) * 4; j < total; j += NT * 4) {
    Four<uint8_t> m{{1, 1, 1, 1}};
    if (mask != nullptr) m.load(mask, j, total);
    Four<T> d;
#pragma unroll
    for (int i = 0; i < 4; ++i) d.v[i] = m.v[i] != 0 ? quiet_nan<T>() : T(0);
    d.store(grad, j, total);
  }
}

template <typename T>
__device__ __forceinline__ void put_policy(const PolicySums& v, T* loss, T* kl, T* cut) {
  const double per = 1.0 / (v.n < 1.0 ? 1.0 : v.n);
  loss[0] = static_cast<T>(v.n >= 0.0 ? v.loss : v.n);
  kl[0] = static_cast<T>(v.kl * per);
  cut[0] = static_cast<T>(v.cut * per);
}

// One pass over the tokens: losses summed, gradients written. Bound by its reads and writes (16384 x 1024
// tokens with a mask and a reference, 285 MB: 50.5 us, 5.6 TB/s; 8.4M ragged tokens with advantages of their
// own, 134 MB: 26.6 us, 5.0 TB/s; workgroups of 128 and 512 threads take 3 and 5 us more, longer runs of tiles by
// one wave 2 to 14 us). Workgroups leave their sums to policy_join_kernel: a last workgroup that sums them after a
// device-wide fence in each cost 160 us more.
template <typename T, int U>
__global__ __launch_bounds__(kThreads) void policy_kernel(PolicyInputs<T> in, Sequences seq,
                                                          double weight, const uint32_t* __restrict__ tokens,
                                                          int count_blocks, const double* __restrict__ weights,
                                                          PolicySums* __restrict__ sums) {
  const int64_t wave = static_cast<int64_t>(blockIdx.x) * kWaves + (threadIdx.x >> 6);
  PolicyPart v;
  __shared__ __attribute__((aligned(16))) int heads[kWaves][256 * U];
  policy_places<T, U>(in, seq, wave * (256 * U), heads[threadIdx.x >> 6], weight, tokens, count_blocks, weights, v);
  const PolicySums all = policy_sums<kThreads>(
      v, unsound(seq, static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x, static_cast<int64_t>(gridDim.x) * kThreads));
  if (threadIdx.x == 0) sums[blockIdx.x] = all;
}

template <typename T>
__global__ __launch_bounds__(kPairThreads) void policy_join_kernel(const PolicySums* __restrict__ sums, int count,
                                                                   T* __restrict__ loss, T* __restrict__ kl,
                                                                   T* __restrict__ cut, const uint8_t* __restrict__ mask,
                                                                   int64_t total, T* __restrict__ grad) {
  double v[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 8
  for (int i = threadIdx.x; i < count; i += kPairThreads) {
    const PolicySums s = sums[i];
    v[0] += s.loss;
    v[1] += s.kl;
    v[2] += s.cut;
    v[3] += s.n;
  }
  block_sums<kPairThreads>(v);
  if (!(v[3] >= 0.0)) void_gradient<kPairThreads>(mask, total, grad);
  if (threadIdx.x == 0) put_policy(PolicySums{v[0], v[1], v[2], v[3]}, loss, kl, cut);
}

// Few tokens in one workgroup: counted, then summed. (Eight sequences, 1616 tokens: 6.8 us, in three launches
// 15 us.)
template <typename T>
__global__ __launch_bounds__(kCountThreads) void policy_small_kernel(PolicyInputs<T> in, Sequences seq, double* weights,
                                                                     T* __restrict__ loss, T* __restrict__ kl,
                                                                     T* __restrict__ cut) {
  double n = static_cast<double>(seq.total);
  if (in.mask != nullptr) {
    n = count_tokens<64>(in.mask, seq, in.reduction, 0, 1, weights);
    __syncthreads();  // (the weights are written)
  }
  const double weight = in.reduction == TI_REDUCE_MEAN ? 1.0 / (n >= 1.0 ? n : 1.0) : 1.0;
  PolicyPart v;
  __shared__ __attribute__((aligned(16))) int heads[kCountThreads / 64][256];
  for (int64_t begin = (threadIdx.x >> 6) * 256; begin < seq.total; begin += kCountThreads / 64 * 256)
    policy_places<T, 1>(in, seq, begin, heads[threadIdx.x >> 6], weight, nullptr, 0, in.mask != nullptr ? weights : nullptr, v);
  const bool bad = unsound(seq, threadIdx.x, kCountThreads);
  const PolicySums all = policy_sums<kCountThreads>(v, bad);
  if (threadIdx.x == 0) put_policy(all, loss, kl, cut);
  if (seq.offsets != nullptr && __syncthreads_or(bad) != 0) void_gradient<kCountThreads>(in.mask, seq.total, in.grad);
}

// grad times g; a g of one leaves it as it is (1.7 us), any other costs a read and a write of it (16384 x 1024
// tokens, 134 MB: 25.4 us, 5.3 TB/s).
template <typename T>
__global__ __launch_bounds__(kThreads) void policy_scale_kernel(T* __restrict__ grad, int64_t total,
                                                                const T* __restrict__ g) {
  const T by = g[0];
  if (by == T(1)) return;
  constexpr int U = 4;
  for (int64_t j0 = static_cast<int64_t>(blockIdx.x) * kThreads * 4 * U; j0 < total;
       j0 += static_cast<int64_t>(gridDim.x) * kThreads * 4 * U) {
    Four<T> d[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t j = j0 + (u * kThreads + threadIdx.x) * 4;
      if (j < total) d[u].load(grad, j, total);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t j = j0 + (u * kThreads + threadIdx.x) * 4;
      // (a masked token's gradient is zero whatever g)
#pragma unroll
      for (int i = 0; i < 4; ++i) d[u].v[i] = d[u].v[i] == T(0) ? T(0) : d[u].v[i] * by;
      if (j < total) d[u].store(grad, j, total);
    }
  }
}

Sequences sequences_of(const SequenceArgs& a) { return Sequences{a.offsets, a.count, a.len, a.total}; }

// At most so many tokens and pairs are one workgroup's, in one launch.
constexpr int64_t kSmall = 4096, kSmallPairs = 32;

// Places a wave takes: fewer where there are few, so that there are waves for the whole GPU. (16384 x 1024 tokens'
// policy loss, a call, with 512 places 63 us, with 1024 66 us; 30000 pairs of 1 to 200 tokens, the preference loss,
// with 512 26.1 us, with 256 30.2 us.)
constexpr int64_t kFew = int64_t{1} << 20;
int64_t tile_places(int64_t total) { return total <= kFew ? 256 : 512; }
int64_t tiles_of(int64_t total) {
  const int64_t places = tile_places(total);
  return (total + places - 1) / places;
}
int64_t blocks_of(int64_t waves) { return waves < kWaves ? 1 : (waves + kWaves - 1) / kWaves; }

// The workspaces: arrays of doubles, one after another.
struct Carve {
  char* at;
  size_t used = 0;
  template <typename T>
  T* take(int64_t n) {
    T* p = reinterpret_cast<T*>(at + used);
    used += static_cast<size_t>(n) * sizeof(T);
    return p;
  }
};
struct PreferenceWork {
  Sum *first, *last, *whole;
  PairPart* parts;
  size_t bytes;
  PreferenceWork(void* work, int64_t total, int64_t sequences) {
    Carve c{static_cast<char*>(work)};
    first = c.take<Sum>(tiles_of(total));
    last = c.take<Sum>(tiles_of(total));
    whole = c.take<Sum>(sequences);
    parts = c.take<PairPart>(kPairBlocks);
    bytes = c.used;
  }
};
struct PolicyWork {
  PolicySums* sums;
  uint32_t* tokens;
  double* weights;
  size_t bytes;
  PolicyWork(void* work, int64_t total, int64_t sequences) {
    Carve c{static_cast<char*>(work)};
    sums = c.take<PolicySums>(blocks_of(tiles_of(total)));
    tokens = c.take<uint32_t>(kCountBlocks);
    weights = c.take<double>(sequences);
    bytes = c.used;
  }
};

}  // namespace

size_t preference_bytes(int64_t total, int64_t sequences) { return PreferenceWork(nullptr, total, sequences).bytes; }

hipError_t preference(const PreferenceArgs& a, void* work) {
  const Sequences seq = sequences_of(a.seq);
  const PreferenceWork w(work, seq.total, seq.count);
  const int64_t places = tile_places(seq.total), pairs = seq.count / 2;
  auto go = [&](auto zero) {
    using T = decltype(zero);
    const PairArgs<T> pa{a.kind, a.average, a.reduction, a.beta, a.smoothing, static_cast<T*>(a.loss),
                         static_cast<T*>(a.chosen), static_cast<T*>(a.rejected), static_cast<T*>(a.slopes)};
    const auto *logps = static_cast<const T*>(a.logps), *ref = static_cast<const T*>(a.ref);
    if (seq.total <= kSmall && pairs <= kSmallPairs) {
      preference_small_kernel<T><<<dim3(1), dim3(kPairThreads), 0, a.stream>>>(logps, ref, a.mask, seq, w.first, w.last, w.whole, pa);
      return hipGetLastError();
    }
    auto sums = places == 256 ? preference_sums_kernel<T, 1> : preference_sums_kernel<T, 2>;
    sums<<<dim3(static_cast<unsigned>(blocks_of(tiles_of(seq.total)))), dim3(kThreads), 0, a.stream>>>(
        logps, ref, a.mask, seq, w.first, w.last, w.whole);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    // (a few lanes a sequence of few tiles, by the mean length: 19999 of 100 tokens and one of 4 million take 95 us,
    // as many tokens spread evenly 26 us)
    const bool few = seq.total / seq.count < places;
    const int64_t each = kPairThreads / 64 * (few ? 8 : 1), want = (pairs + each - 1) / each;
    const int64_t blocks = want < kPairBlocks ? want : kPairBlocks;
    auto kernel = few ? preference_pairs_kernel<T, 4> : preference_pairs_kernel<T, 32>;
    kernel<<<dim3(static_cast<unsigned>(blocks)), dim3(kPairThreads), 0, a.stream>>>(seq, static_cast<int>(places), w.first,
                                                                                    w.last, w.whole, pa, w.parts);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess || blocks == 1 || a.reduction == TI_REDUCE_NONE) return e;
    preference_mean_kernel<T><<<dim3(1), dim3(kPairThreads), 0, a.stream>>>(
        w.parts, static_cast<int>(blocks), a.reduction == TI_REDUCE_MEAN ? 1.0 / static_cast<double>(pairs) : 1.0, pa.loss,
        pa.slopes, seq.count);
    return hipGetLastError();
  };
  return a.dtype == TI_F32 ? go(float{}) : go(double{});
}

hipError_t preference_grad(const SequenceArgs& s, const uint8_t* mask, const void* slopes, const void* g, int per_pair,
                           void* grad, int dtype, hipStream_t stream) {
  auto go = [&](auto zero) {
    using T = decltype(zero);
    auto kernel = tile_places(s.total) == 256 ? preference_grad_kernel<T, 1> : preference_grad_kernel<T, 2>;
    kernel<<<dim3(static_cast<unsigned>(blocks_of(tiles_of(s.total)))), dim3(kThreads), 0, stream>>>(
        mask, sequences_of(s), static_cast<const T*>(slopes), static_cast<const T*>(g), per_pair,
        static_cast<T*>(grad));
    return hipGetLastError();
  };
  return dtype == TI_F32 ? go(float{}) : go(double{});
}

size_t policy_bytes(int64_t total, int64_t sequences) { return PolicyWork(nullptr, total, sequences).bytes; }

hipError_t policy(const PolicyArgs& a, void* work) {
  const Sequences seq = sequences_of(a.seq);
  const PolicyWork w(work, seq.total, seq.count);
  auto go = [&](auto zero) {
    using T = decltype(zero);
    const PolicyInputs<T> in{static_cast<const T*>(a.logps), static_cast<const T*>(a.old), static_cast<const T*>(a.adv),
                             static_cast<const T*>(a.ref), a.mask, a.adv_each, a.reduction, Clip<T>(a.lo, a.hi),
                             static_cast<T>(a.kl_coef), static_cast<T*>(a.grad)};
    auto *loss = static_cast<T*>(a.loss), *kl = static_cast<T*>(a.kl), *cut = static_cast<T*>(a.cut);
    if (seq.total <= kSmall && seq.count <= 2 * kSmallPairs) {
      policy_small_kernel<T><<<dim3(1), dim3(kCountThreads), 0, a.stream>>>(in, seq, w.weights, loss, kl, cut);
      return hipGetLastError();
    }
    const bool mean = a.reduction == TI_REDUCE_MEAN, by_sequence = a.reduction == TI_REDUCE_SEQUENCES;
    int blocks = 0;
    if (seq.total > 0 && a.mask != nullptr && (mean || by_sequence)) {
      // masked sequences counted by as many threads as their mean length asks for (20000 of 1 to 600 tokens, the
      // policy loss: by 8 threads each 35.7 us, by 64 41.7 us; 8000 of 1 to 2000: 49.3 and 45.2 us), which a sequence
      // far longer than the mean waits for (20000 of 200 tokens and one of 131072: 321 us, as many tokens spread
      // evenly 29 us; 19999 of 100 and one of 4 million: 9.0 ms and 38 us); else the places in turn
      const int64_t length = seq.total / seq.count;
      const int lanes = mean ? 64 : (length >= 32768 ? kCountThreads : (length >= 512 ? 64 : 8));
      const int64_t want = mean ? (seq.total + 16383) / 16384 : (seq.count + kCountThreads / lanes - 1) / (kCountThreads / lanes);
      const int64_t most = mean ? kCountBlocks : kWeightBlocks;
      blocks = static_cast<int>(want > most ? most : (want + 3) / 4 * 4);  // (a multiple of four)
      auto count = lanes == kCountThreads ? policy_count_kernel<kCountThreads>
                                          : (lanes == 64 ? policy_count_kernel<64> : policy_count_kernel<8>);
      count<<<dim3(blocks), dim3(kCountThreads), 0, a.stream>>>(a.mask, seq, a.reduction, w.tokens, w.weights);
      if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    const double weight = mean && seq.total > 0 ? 1.0 / static_cast<double>(seq.total) : 1.0;
    const int64_t tiles = blocks_of(tiles_of(seq.total));
    auto kernel = tile_places(seq.total) == 256 ? policy_kernel<T, 1> : policy_kernel<T, 2>;
    kernel<<<dim3(static_cast<unsigned>(tiles)), dim3(kThreads), 0, a.stream>>>(
        in, seq, weight, mean && blocks > 0 ? w.tokens : nullptr, blocks, blocks > 0 ? w.weights : nullptr, w.sums);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    policy_join_kernel<T><<<dim3(1), dim3(kPairThreads), 0, a.stream>>>(w.sums, static_cast<int>(tiles), loss, kl, cut, in.mask,
                                                                         seq.total, in.grad);
    return hipGetLastError();
  };
  return a.dtype == TI_F32 ? go(float{}) : go(double{});
}

hipError_t policy_scale(void* grad, int64_t total, const void* g, int dtype, hipStream_t stream) {
  const int64_t want = (total + 16 * kThreads - 1) / (16 * kThreads);
  const unsigned blocks = static_cast<unsigned>(want > 1024 ? 1024 : want);
  auto go = [&](auto zero) {
    using T = decltype(zero);
    policy_scale_kernel<T><<<dim3(blocks), dim3(kThreads), 0, stream>>>(static_cast<T*>(grad), total, static_cast<const T*>(g));
    return hipGetLastError();
  };
  return dtype == TI_F32 ? go(float{}) : go(double{});
}

}  // namespace ti
