// gfx950 kernels for log probabilities (plh_logprobs): of each row the
// normaliser lse = m + log(sum exp(x - m)), the chosen token's x - lse and rank,
// and the n best tokens.
//
// One pass over the logits.  A workgroup walks one segment of a row in chunks of
// kLpChunk tokens, the next chunk's loads in flight while it works on one.  In
// the walk every thread keeps its own running maximum and (float64) sum, and
// every wave its own list of candidates for the n best with a threshold that n
// tokens of the list reach, so that the walk has no barrier: a chunk of a wave
// (1024 tokens) whose 64 lane maxima all lie at or below the threshold costs one
// ballot; where n of them lie above it, the n-th largest is the new threshold.
// At the end the waves cut their lists to n and the workgroup ranks what reaches
// the best of the waves' thresholds.  Rows shared out over several segments leave
// (m, sum, rank count, n candidates) each for a second launch.
//
// Tokens of -inf never enter a list: a row with fewer than n others fills up with
// its lowest tokens that are not listed (under a grammar's mask most tokens are
// -inf).  All counts are integers and all sums have a fixed order.
//
// Bound by the read of the logits.
#include "plh_device.h"
#include "plh_kernels.h"

#include <algorithm>

namespace plh {

namespace {

constexpr int kLpChunk = 8192;
constexpr int kVals = kLpChunk / kThreads;  // tokens of a chunk per thread, in groups of four
constexpr int kList = 256;                  // candidate slots of a wave
constexpr int kMergeList = 1024;            // candidates that the second launch ranks in LDS

// Order keys: larger value, larger key; -0 and 0 alike, every NaN the largest.
template <typename T>
struct Order;
template <>
struct Order<float> {
  typedef uint32_t K;
  static constexpr int kBits = 32;
  static constexpr K kNegInf = 0x007fffffu;
  static __device__ __forceinline__ K key(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return x != x ? 0xffffffffu : (u >> 31) ? ~u : (u | 0x80000000u);
  }
  static __device__ __forceinline__ float value(K k) {
    return k == 0xffffffffu ? NAN : __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k);
  }
};
template <>
struct Order<double> {
  typedef uint64_t K;
  static constexpr int kBits = 64;
  static constexpr K kNegInf = 0x000fffffffffffffull;
  static __device__ __forceinline__ K key(double x) { return x != x ? ~0ull : key_of(x); }
  static __device__ __forceinline__ double value(K k) { return k == ~0ull ? (double)NAN : val_of_key(k); }
};

__device__ __forceinline__ double exp_term(float d) {
  return (double)__builtin_amdgcn_exp2f(d * 1.44269504088896340736f);
}
__device__ __forceinline__ double exp_term(double d) { return exp(d); }

template <typename K>
__device__ __forceinline__ bool before(K ka, int ia, K kb, int ib) {
  return ka > kb || (ka == kb && ia < ib);
}

// The largest t that at least n of the wave's keys reach (n of them do), or some
// t that exactly n reach.
template <typename T, int R>
__device__ __forceinline__ typename Order<T>::K nth_key(const typename Order<T>::K (&k)[R], int n) {
  typedef typename Order<T>::K K;
  K t = 0;
  for (int b = Order<T>::kBits - 1; b >= 0; --b) {
    const K trial = t | ((K)1 << b);
    int c = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) c += __popcll(__ballot(k[r] >= trial));
    if (c >= n) t = trial;
    if (c == n) break;
  }
  return t;
}

// A wave's candidate list in LDS.
template <typename T>
struct List {
  typename Order<T>::K* key;
  int* id;
};

// Cuts a list of len >= n entries to its n first in the order; returns the
// threshold that exactly these reach among themselves.
template <typename T>
__device__ typename Order<T>::K prune(const List<T>& l, int len, int n) {
  typedef typename Order<T>::K K;
  constexpr int R = kList / kWave;
  K k[R];
  int id[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = r * kWave + lane();
    k[r] = i < len ? l.key[i] : 0;
    id[r] = i < len ? l.id[i] : INT_MAX;
  }
  const K t = nth_key<T, R>(k, n);
  int above = 0, reach = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    above += __popcll(__ballot(k[r] > t));
    reach += __popcll(__ballot(k[r] >= t));
  }
  int last = INT_MAX;  // of the tokens at t itself, the lowest ids
  if (reach > n) {
    for (int b = 30; b >= 0; --b) {
      const int trial = last & ~(1 << b);
      int c = above;
#pragma unroll
      for (int r = 0; r < R; ++r) c += __popcll(__ballot(k[r] == t && id[r] <= trial));
      if (c >= n) last = trial;
    }
  }
  __builtin_amdgcn_wave_barrier();
  int at = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool keep = k[r] > t || (k[r] == t && id[r] <= last);
    const uint64_t m = __ballot(keep);
    if (keep) {
      const int p = at + __popcll(m & ((1ull << lane()) - 1));
      l.key[p] = k[r];
      l.id[p] = id[r];
    }
    at += __popcll(m);
  }
  __builtin_amdgcn_wave_barrier();
  return t;
}

// What a segment leaves for the second launch, before its n candidates' keys and
// ids.
struct Part {
  double m, s;
  int above, count;
};

template <typename T>
__host__ __device__ constexpr size_t part_bytes(int n) {
  return sizeof(Part) + ((size_t)n * (sizeof(T) + 4) + 7) / 8 * 8;
}

template <typename T>
struct PartView {
  Part* part;
  typename Order<T>::K* key;
  int* id;
};

template <typename T>
__device__ __forceinline__ PartView<T> part_of(const LogprobsArgs& a, int row, int seg) {
  typedef typename Order<T>::K K;
  char* p = static_cast<char*>(a.ws) + ((size_t)row * a.segs + seg) * part_bytes<T>(a.n);
  K* key = reinterpret_cast<K*>(p + sizeof(Part));
  return PartView<T>{reinterpret_cast<Part*>(p), key, reinterpret_cast<int*>(key + a.n)};
}

// The log probability of x under a row of maximum m and sum s.
template <typename T>
__device__ __forceinline__ T log_prob(double x, double m, double s) {
  if (m == -INFINITY && s == 0.0) return (T)-INFINITY;  // nothing but -inf in the row
  return (T)((x - m) - log(s));
}

template <typename T>
__device__ __forceinline__ void write_chosen(const LogprobsArgs& a, int row, double m, double s, int above) {
  if (a.ids == nullptr || threadIdx.x != 0) return;
  const int id = a.ids[row];
  const bool ok = (unsigned)id < (unsigned)a.V;
  static_cast<T*>(a.lp)[row] =
      ok ? log_prob<T>((double)static_cast<const T*>(a.x)[(int64_t)row * a.ld + id], m, s) : (T)NAN;
  a.rank[row] = ok ? above + 1 : 0;
}

template <typename T>
__device__ __forceinline__ void write_top(const LogprobsArgs& a, int row, int r, typename Order<T>::K k, int id,
                                          double m, double s) {
  a.top_ids[(int64_t)row * a.n + r] = id;
  static_cast<T*>(a.top_lp)[(int64_t)row * a.n + r] = log_prob<T>((double)Order<T>::value(k), m, s);
}

// Entries `have` .. n-1 of a row with `have` tokens above -inf, all of them in
// ids[]: its lowest tokens that are not among them.
template <typename T>
__device__ void fill_top(const LogprobsArgs& a, int row, const int* ids, int have, double m, double s, int* red) {
  const int t = threadIdx.x;  // n + have < 2 * kMaxTop <= kThreads
  bool free_token = t < a.V && t < a.n;
  for (int j = 0; j < have; ++j) free_token = free_token && ids[j] != t;
  // of n tokens and those listed among them, at least n - have are free
  int total;
  const int at = have + block_excl_scan<int>(free_token ? 1 : 0, red, &total);
  if (free_token && at < a.n) write_top<T>(a, row, at, Order<T>::kNegInf, t, m, s);
}

typedef float f32x4e __attribute__((ext_vector_type(4))) __attribute__((aligned(4)));
typedef double f64x2e __attribute__((ext_vector_type(2))) __attribute__((aligned(8)));

__device__ __forceinline__ void load4(const float* p, float* v) {
  const f32x4e q = *reinterpret_cast<const f32x4e*>(p);
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = q[e];
}
__device__ __forceinline__ void load4(const double* p, double* v) {
  const f64x2e q = *reinterpret_cast<const f64x2e*>(p), r = *reinterpret_cast<const f64x2e*>(p + 2);
  v[0] = q[0], v[1] = q[1], v[2] = r[0], v[3] = r[1];
}

// The thread's tokens of the chunk at c0: group g holds tokens c0 + 4 (g *
// kThreads + thread) .. + 3; those past the row's end read as -inf.
template <typename T>
__device__ __forceinline__ void load_chunk(const T* x, int64_t c0, int V, T (&v)[kVals]) {
#pragma unroll
  for (int g = 0; g < kVals / 4; ++g) {
    const int64_t t = c0 + 4 * (g * kThreads + (int)threadIdx.x);
    if (t + 4 <= V) {
      load4(x + t, &v[4 * g]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * g + e] = t + e < V ? x[t + e] : (T)-INFINITY;
    }
  }
}

// TOP: n > 0.
template <typename T, bool TOP>
__global__ __launch_bounds__(kThreads) void k_logprobs(LogprobsArgs a) {
  typedef Order<T> O;
  typedef typename O::K K;
  __shared__ K lkey[TOP ? kWaves * kList : 1];
  __shared__ int lid[TOP ? kWaves * kList : 1];
  __shared__ double redd[kWaves];
  __shared__ int redi[kWaves];
  __shared__ K wthr[kWaves];
  __shared__ int wlen[kWaves];
  const int seg = blockIdx.x;
  for (int row = blockIdx.y; row < a.B; row += gridDim.y) {
    const T* x = static_cast<const T*>(a.x) + (int64_t)row * a.ld;
    const int64_t first = (int64_t)seg * a.seg_chunks * kLpChunk;
    const int64_t end = min((int64_t)a.V, first + (int64_t)a.seg_chunks * kLpChunk);
    T v[kVals], next[kVals];
    load_chunk(x, first, a.V, next);
    int chosen = -1;
    K ck = 0;
    if (a.ids != nullptr) {
      chosen = a.ids[row];
      if ((unsigned)chosen < (unsigned)a.V) ck = O::key(x[chosen]);
      else chosen = -1;
    }
    T m = (T)-INFINITY;
    double s = 0.0;
    int above = 0, len = 0;
    K thr = O::kNegInf;  // tokens at or below it are out of the wave's list
    const List<T> list{lkey + (TOP ? wave() * kList : 0), lid + (TOP ? wave() * kList : 0)};
    for (int64_t c0 = first; c0 < end; c0 += kLpChunk) {
#pragma unroll
      for (int i = 0; i < kVals; ++i) v[i] = next[i];
      if (c0 + kLpChunk < end) load_chunk(x, c0 + kLpChunk, a.V, next);
      T mt = v[0];
#pragma unroll
      for (int i = 1; i < kVals; ++i) mt = fmax(mt, v[i]);
      const T mn = fmax(m, mt);
      const T M = mn == (T)-INFINITY ? (T)0 : mn;  // -inf - M is -inf
      if (!(mn == m)) s *= exp((double)m - (double)M);
      m = mn;
#pragma unroll
      for (int i = 0; i < kVals; ++i) s += exp_term(v[i] - M);
      K k[kVals], km = 0;
#pragma unroll
      for (int i = 0; i < kVals; ++i) {
        k[i] = O::key(v[i]);
        km = k[i] > km ? k[i] : km;
      }
      const int64_t t0 = c0 + 4 * (int)threadIdx.x;
      if (chosen >= 0) {
#pragma unroll
        for (int i = 0; i < kVals; ++i) {
          const int64_t t = t0 + 4 * (i / 4) * kThreads + i % 4;
          above += k[i] > ck || (k[i] == ck && t < chosen);
        }
      }
      if constexpr (TOP) {
        const int lanes = __popcll(__ballot(km > thr));
        if (lanes == 0) continue;
        // at least n tokens of the chunk reach the n-th of the lane maxima
        const bool enough = lanes >= a.n;
        K reach = thr + 1;  // thr is below some key here
        if (enough) {
          const K one[1] = {km};
          reach = nth_key<T, 1>(one, a.n);
        }
        bool cut = enough;
#pragma unroll
        for (int i = 0; i < kVals; ++i) {
          uint64_t in = __ballot(k[i] >= reach);
          if (in == 0) continue;
          if (len + __popcll(in) > kList) {
            reach = prune(list, len, a.n);
            len = a.n;
            cut = true;
            in = __ballot(k[i] >= reach);
          }
          if (k[i] >= reach) {
            const int p = len + __popcll(in & ((1ull << lane()) - 1));
            list.key[p] = k[i];
            list.id[p] = (int)(t0 + 4 * (i / 4) * kThreads + i % 4);
          }
          len += __popcll(in);
        }
        if (cut) thr = reach;  // n listed tokens reach it, with lower ids than any that follow
      }
    }
    // the segment's maximum and sum
    const double mb = block_max((double)m, redd);
    const double Mb = mb == -INFINITY ? 0.0 : mb;
    const double sb = block_sum(s * exp((double)m - Mb), redd);
    const int ab = block_sum(above, redi);
    const PartView<T> pv = part_of<T>(a, row, seg);
    if (a.segs == 1) write_chosen<T>(a, row, mb, sb, ab);
    int count = 0;
    if constexpr (TOP) {
      if (len >= a.n) {
        thr = prune(list, len, a.n);
        len = a.n;
      } else {
        thr = 0;
      }
      if (lane() == 0) {
        wthr[wave()] = thr;
        wlen[wave()] = len;
      }
      wg_barrier();
      K best = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) best = wthr[w] > best ? wthr[w] : best;
      // one entry per thread (len <= n <= 64); those below `best` are not among the n
      const bool in = lane() < len && list.key[lane()] >= best;
      const K k = in ? list.key[lane()] : 0;
      const int id = in ? list.id[lane()] : 0;
      wg_barrier();
      const int at = block_excl_scan<int>(in ? 1 : 0, redi, &count);
      if (in) {
        lkey[at] = k;
        lid[at] = id;
      }
      wg_barrier();
      if (in) {
        int r = 0;
        for (int j = 0; j < count; ++j) r += before<K>(lkey[j], lid[j], k, id);
        if (r < a.n) {
          if (a.segs == 1) {
            write_top<T>(a, row, r, k, id, mb, sb);
          } else {
            pv.key[r] = k;
            pv.id[r] = id;
          }
        }
      }
      if (a.segs == 1 && count < a.n) fill_top<T>(a, row, lid, count, mb, sb, redi);
      wg_barrier();  // the lists are read before the next row writes them
    }
    if (a.segs > 1 && threadIdx.x == 0) *pv.part = Part{mb, sb, ab, min(count, a.n)};
  }
}

// One workgroup per row joins its segments.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_logprobs_merge(LogprobsArgs a) {
  typedef Order<T> O;
  typedef typename O::K K;
  __shared__ K lkey[kMergeList];
  __shared__ int lid[kMergeList];
  __shared__ double redd[kWaves];
  __shared__ int redi[kWaves];
  __shared__ K redk[kWaves];
  __shared__ int fill;
  for (int row = blockIdx.x; row < a.B; row += gridDim.x) {
    if (threadIdx.x == 0) fill = 0;
    double m = -INFINITY, s = 0.0;
    int above = 0, have = 0;
    K best = 0;
    for (int g = threadIdx.x; g < a.segs; g += kThreads) {
      const PartView<T> pv = part_of<T>(a, row, g);
      const Part p = *pv.part;
      const double mn = fmax(m, p.m), M = mn == -INFINITY ? 0.0 : mn;
      s = s * exp(m - M) + p.s * exp(p.m - M);
      m = mn;
      above += p.above;
      have += p.count;
      if (a.n > 0 && p.count == a.n) {
        const K k = pv.key[a.n - 1];
        best = k > best ? k : best;
      }
    }
    const double mb = block_max(m, redd);
    const double Mb = mb == -INFINITY ? 0.0 : mb;
    const double sb = block_sum(s * exp(m - Mb), redd);
    above = block_sum(above, redi);
    write_chosen<T>(a, row, mb, sb, above);
    if (a.n == 0) continue;
    have = min(block_sum(have, redi), a.n);
    best = block_max(best, redk);
    const int64_t entries = (int64_t)a.segs * a.n;
    for (int64_t e = threadIdx.x; e < entries; e += kThreads) {
      const PartView<T> pv = part_of<T>(a, row, (int)(e / a.n));
      const int j = (int)(e % a.n);
      if (j < pv.part->count && pv.key[j] >= best) {
        const int p = lds_fetch_add(&fill, 1);
        if (p < kMergeList) {
          lkey[p] = pv.key[j];
          lid[p] = pv.id[j];
        }
      }
    }
    wg_barrier();
    const int count = fill;
    if (count <= kMergeList) {
      for (int i = threadIdx.x; i < count; i += kThreads) {
        int r = 0;
        for (int j = 0; j < count; ++j) r += before<K>(lkey[j], lid[j], lkey[i], lid[i]);
        if (r < a.n) write_top<T>(a, row, r, lkey[i], lid[i], mb, sb);
      }
      if (have < a.n) fill_top<T>(a, row, lid, have, mb, sb, redi);
    } else {
      // very many like values over very many segments: the n first one by one
      K lk = ~(K)0;
      int li = -1;
      for (int r = 0; r < a.n; ++r) {
        K bk = 0;
        int bi = INT_MAX;
        for (int64_t e = threadIdx.x; e < entries; e += kThreads) {
          const PartView<T> pv = part_of<T>(a, row, (int)(e / a.n));
          const int j = (int)(e % a.n);
          if (j >= pv.part->count) continue;
          const K k = pv.key[j];
          const int id = pv.id[j];
          if (before<K>(lk, li, k, id) && before<K>(k, id, bk, bi)) bk = k, bi = id;
        }
        const K k = block_max(bk, redk);
        const int id = block_min(bk == k ? bi : INT_MAX, redi);
        if (threadIdx.x == 0) write_top<T>(a, row, r, k, id, mb, sb);
        lk = k, li = id;
      }
    }
    wg_barrier();
  }
}

template <typename T>
hipError_t launch_t(const LogprobsArgs& a, hipStream_t s) {
  const dim3 grid(a.segs, std::min(a.B, 65535));
  if (a.n > 0) hipLaunchKernelGGL((k_logprobs<T, true>), grid, dim3(kThreads), 0, s, a);
  else hipLaunchKernelGGL((k_logprobs<T, false>), grid, dim3(kThreads), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.segs == 1) return e;
  hipLaunchKernelGGL((k_logprobs_merge<T>), dim3(a.B), dim3(kThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace

// Segments: as many workgroups as four per compute unit, a whole chunk or more
// each.
size_t plan_logprobs(LogprobsArgs& a, bool f64, int num_cu, bool one_launch) {
  const int64_t chunks = ((int64_t)a.V + kLpChunk - 1) / kLpChunk, target = 4 * (int64_t)num_cu;
  const int64_t each = one_launch ? chunks : std::min(chunks, (a.B * chunks + target - 1) / target);
  a.seg_chunks = (int)each;
  a.segs = (int)((chunks + each - 1) / each);
  return a.segs == 1 ? 0 : (size_t)a.B * a.segs * (f64 ? part_bytes<double>(a.n) : part_bytes<float>(a.n));
}

hipError_t launch_logprobs(const LogprobsArgs& a, bool f64, hipStream_t s) {
  return f64 ? launch_t<double>(a, s) : launch_t<float>(a, s);
}

}  // namespace plh
