// gfx950 kernels for log probabilities (plh_logprobs): of each row the
// normaliser lse = m + log(sum exp(x - m)), the chosen token's x - lse and rank,
// and the n best tokens.
//
// One pass over the logits.  A workgroup walks one segment of a row in chunks of
// 32 KB (8192 float32 tokens), the next chunk's loads in flight while it works on one.  In
// the walk every thread keeps its own running maximum and (float64) sum, and
// every wave its own list of candidates for the n best, with a threshold that n
// listed tokens reach.  The threads' maxima over the first two chunks give the
// first threshold (about their n-th largest); from there on the walk has no barrier: a
// chunk of a wave (1024 float32 tokens) whose 64 lane maxima all lie at or below the
// threshold costs one ballot, and where n of them lie above it, the n-th largest is
// the new one.  At the end the workgroup ranks what reaches the best of the waves'
// thresholds.  Rows shared out over several segments leave (m, sum, rank count, n
// candidates) each for a second launch.
//
// Tokens of -inf never enter a list: a row with fewer than n others fills up with
// its lowest tokens that are not listed (under a grammar's mask most tokens are
// -inf).  All counts are integers and all sums have a fixed order.
//
// Bound by the read of the logits, where there is no list: 2048 x 32 000 57 us, 4.6
// TB/s.  The n best cost the chains at the start and end of each segment and the
// second launch: 256 x 128 256 33 us without, 46-47 us with 20 of them
// (97 us with a threshold searched by every wave in every chunk).
#include "plh_fast.h"
#include "plh_kernels.h"

#include <algorithm>

namespace plh {

namespace {

// Tokens of a chunk per thread, in groups of four: 64 bytes.
template <typename T>
constexpr int kValsOf = 64 / sizeof(T);
template <typename T>
constexpr int kChunkOf = kValsOf<T> * kThreads;
constexpr int kList = 128;                  // candidate slots of a wave: twice the most that are asked for
static_assert(kList >= 2 * kMaxTop && kWaves * kList >= kThreads, "n listed and n of a chunk; a key per thread");
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

// exp(d) for d <= 0 as a term of a row's sum; NaN for what is not (a NaN, or
// inf - inf).
__device__ __forceinline__ double exp_term(float d, const double*) {
  return (double)__builtin_amdgcn_exp2f(d * 1.44269504088896340736f);
}
__device__ __forceinline__ double exp_term(double d, const double* tab) {
  return d <= 0.0 ? exp_neg_term(d, tab) : (double)NAN;
}

// The factor that takes a sum from the maximum m to M >= m.
__device__ __forceinline__ double rescale(double m, double M, const double* tab) {
  return m < M ? exp_neg_term(m - M, tab) : 1.0;
}

template <typename K>
__device__ __forceinline__ bool before(K ka, int ia, K kb, int ib) {
  return ka > kb || (ka == kb && ia < ib);
}

template <typename K, int R>
__device__ __forceinline__ int count_ge(const K (&k)[R], K t) {
  int c = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) c += __popcll(__ballot(k[r] >= t));
  return c;
}

// The largest t that at least n of the wave's keys reach (n of them do), or some
// t that n to `most` of them reach.  Down from the largest key in growing steps (the
// first about a twelfth of a value), then by halves.
template <typename T, int R>
__device__ __forceinline__ typename Order<T>::K nth_key(const typename Order<T>::K (&k)[R], int n, int most) {
  typedef typename Order<T>::K K;
  K top = k[0];
#pragma unroll
  for (int r = 1; r < R; ++r) top = k[r] > top ? k[r] : top;
  top = wave_max(top);
  K lo = top, step = (K)1 << (Order<T>::kBits == 32 ? 20 : 49);
  int c = count_ge<K, R>(k, lo);
  while (c < n) {
    top = lo;
    lo = step != 0 && lo > step ? lo - step : 0;  // all keys reach 0
    step <<= 1;
    c = count_ge<K, R>(k, lo);
  }
  while (c > most && top - lo > 1) {
    const K mid = lo + (top - lo) / 2;
    const int m = count_ge<K, R>(k, mid);
    if (m >= n) lo = mid, c = m;
    else top = mid;
  }
  return lo;
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
__device__ __forceinline__ typename Order<T>::K prune(const List<T>& l, int len, int n) {
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
  const K t = nth_key<T, R>(k, n, n);
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

// Calls f(rank, key, id) for each of the count entries (in LDS), a thread or a
// group of threads of the workgroup each: 8 up to 64 entries, 4 up to 128, ...
template <typename K, class F>
__device__ __forceinline__ void rank_list(const K* key, const int* id, int count, const F& f) {
  int each = 8;
  while (each > 1 && count * each > kThreads) each >>= 1;
  const int part = (int)threadIdx.x & (each - 1);
  for (int i = (int)threadIdx.x / each; i < count; i += kThreads / each) {
    const K k = key[i];
    const int t = id[i];
    int r = 0;
#pragma unroll 4
    for (int j = part; j < count; j += each) r += before<K>(key[j], id[j], k, t);
    for (int d = 1; d < each; d <<= 1) r += __shfl_xor(r, d);
    if (part == 0) f(r, k, t);
  }
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
  if (m == -INFINITY && s == s) return (T)-INFINITY;  // nothing but -inf in the row
  return (T)((x - m) - log(s));
}

// The chosen token's answers, x its logit (read ahead of the sums), id -1 for an id
// outside the vocabulary.
template <typename T>
__device__ __forceinline__ void write_chosen(const LogprobsArgs& a, int row, int id, T x, double m, double s,
                                             int above) {
  if (a.ids == nullptr || threadIdx.x != 0) return;
  static_cast<T*>(a.lp)[row] = id >= 0 ? log_prob<T>((double)x, m, s) : (T)NAN;
  a.rank[row] = id >= 0 ? above + 1 : 0;
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
__device__ __forceinline__ void load_chunk(const T* x, int64_t c0, int V, T (&v)[kValsOf<T>]) {
  constexpr int kVals = kValsOf<T>, kLpChunk = kChunkOf<T>;
  const T* p = x + c0;  // uniform
  const int t = 4 * (int)threadIdx.x, left = (int)min((int64_t)kLpChunk, V - c0);
  if (left == kLpChunk) {
#pragma unroll
    for (int g = 0; g < kVals / 4; ++g) load4(p + 4 * g * kThreads + t, &v[4 * g]);
  } else {
#pragma unroll
    for (int g = 0; g < kVals / 4; ++g) {
      if (t + 4 * g * kThreads + 4 <= left) {
        load4(p + 4 * g * kThreads + t, &v[4 * g]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = t + 4 * g * kThreads + e;
          v[4 * g + e] = i < left ? p[i] : (T)-INFINITY;
        }
      }
    }
  }
}

// TOP: n > 0.
template <typename T, bool TOP>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(4))) void
k_logprobs(LogprobsArgs a) {
  typedef Order<T> O;
  typedef typename O::K K;
  constexpr int kVals = kValsOf<T>, kLpChunk = kChunkOf<T>;
  __shared__ K lkey[TOP ? kWaves * kList : 1];
  __shared__ int lid[TOP ? kWaves * kList : 1];
  __shared__ double redm[kWaves], redd[kWaves];
  __shared__ int redi[kWaves];
  __shared__ K wthr[kWaves], sthr;
  __shared__ int wlen[kWaves];
  __shared__ int fill;
  __shared__ double tabs[kWaves * kWave];
  double* tab = tabs + wave() * kWave;
  init_exp_table_wave(tab);
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
    const T cv = chosen >= 0 ? O::value(ck) : (T)0;
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
      s *= rescale((double)m, (double)M, tab);
      m = mn;
#pragma unroll
      for (int g = 0; g < kVals; g += 4) {
#pragma unroll
        for (int i = g; i < g + 4; ++i) s += exp_term(v[i] - M, tab);
        __builtin_amdgcn_sched_barrier(0);  // four terms at a time in registers
      }
      const uint32_t t0 = (uint32_t)c0 + 4 * threadIdx.x;
      const auto token = [&](int i) { return t0 + 4 * (i / 4) * kThreads + i % 4; };
      // a NaN, which the maxima pass over, shows in the sum from then on
      const bool nan = s != s;
      if (chosen >= 0 && __ballot(!(mt < cv) || nan) != 0) {
#pragma unroll
        for (int i = 0; i < kVals; ++i) {
          const K k = O::key(v[i]);
          above += k > ck || (k == ck && token(i) < (uint32_t)chosen);
        }
      }
      if constexpr (TOP) {
        const bool start = c0 == first;  // uniform
        // the start's threshold holds n tokens of the first two chunks, so that only
        // from the third on a like one is behind them
        const K pass = c0 - first <= kLpChunk && thr > O::kNegInf ? thr : thr + 1;
        const K one[1] = {O::key(mt)};
        if (!start && (pass == 0 || __ballot(one[0] >= pass || nan) == 0)) continue;  // (0: behind n NaNs)
        K reach;
        if (start) {
          // n tokens reach about the n-th of the threads' maxima over this chunk and
          // the next
          T mx = mt;
          if (c0 + kLpChunk < end) {
#pragma unroll
            for (int i = 0; i < kVals; ++i) mx = fmax(mx, next[i]);
          }
          lkey[threadIdx.x] = O::key(mx);
          wg_barrier();
          if (wave() == 0) {
            K all[kWaves];
            int c = 0;
#pragma unroll
            for (int r = 0; r < kWaves; ++r) {
              all[r] = lkey[r * kWave + lane()];
              c += __popcll(__ballot(all[r] > O::kNegInf));
            }
            const K t = c >= a.n ? nth_key<T, kWaves>(all, a.n, a.n + a.n / 4) : O::kNegInf;
            if (lane() == 0) sthr = t;
          }
          wg_barrier();
          thr = sthr;
          reach = thr > O::kNegInf ? thr : thr + 1;
          if (__ballot(one[0] >= reach || nan) == 0) continue;
        } else {
          reach = pass;
          if (__popcll(__ballot(one[0] >= pass)) >= a.n) {
            // the same for a wave, where a row rises (all 64 lanes reach any smaller key)
            const K t = nth_key<T, 1>(one, a.n, a.n);
            reach = t > pass ? t : pass;
            thr = reach;
          }
        }
        if (__ballot(nan) == 0) {
          // mostly a lane or two have such tokens: no keys but for them
          const T floor = O::value(reach);
          if (len + kVals * __popcll(__ballot(mt >= floor)) <= kList) {
#pragma unroll
            for (int i = 0; i < kVals; ++i) {
              const uint64_t in = __ballot(v[i] >= floor);
              if (in == 0) continue;
              if (v[i] >= floor) {
                const int p = len + __popcll(in & ((1ull << lane()) - 1));
                list.key[p] = O::key(v[i]);
                list.id[p] = (int)token(i);
              }
              len += __popcll(in);
            }
            continue;
          }
        }
        K k[kVals];
#pragma unroll
        for (int i = 0; i < kVals; ++i) k[i] = O::key(v[i]);
        if (len + count_ge<K, kVals>(k, reach) > kList) {
          if (len >= a.n) {
            const K t = prune(list, len, a.n);
            len = a.n;
            if (t >= reach) {
              thr = t;
              if (t == ~(K)0) continue;
              reach = t + 1;
            }
          }
          if (len + count_ge<K, kVals>(k, reach) > kList) {
            // many like values, or a chunk that rises: exactly n of it, of like ones
            // the first (n are there: else they would fit)
            reach = nth_key<T, kVals>(k, a.n, a.n);
            thr = reach;
            uint32_t last = UINT_MAX;
            const auto count = [&](uint32_t id) {
              int c = 0;
#pragma unroll
              for (int i = 0; i < kVals; ++i) c += __popcll(__ballot(k[i] > reach || (k[i] == reach && token(i) <= id)));
              return c;
            };
            for (int b = 31; b >= 0; --b) {
              const uint32_t trial = last & ~(1u << b);
              if (count(trial) >= a.n) last = trial;
            }
#pragma unroll
            for (int i = 0; i < kVals; ++i) k[i] = k[i] == reach && token(i) > last ? 0 : k[i];
          }
        }
#pragma unroll
        for (int i = 0; i < kVals; ++i) {
          const uint64_t in = __ballot(k[i] >= reach);
          if (in == 0) continue;
          if (k[i] >= reach) {
            const int p = len + __popcll(in & ((1ull << lane()) - 1));
            list.key[p] = k[i];
            list.id[p] = (int)token(i);
          }
          len += __popcll(in);
        }
      }
    }
    // the segment's maximum, sum and rank count, and what its waves' lists hold: two
    // rounds through LDS
    const double mw = wave_max((double)m);
    if (threadIdx.x == 0) fill = 0;
    if (lane() == 0) {
      redm[wave()] = mw;
      wthr[wave()] = thr;
      wlen[wave()] = len;
    }
    wg_barrier();
    double mb = redm[0];
    K best = wthr[0];  // n listed tokens reach it
    int listed = wlen[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
      mb = fmax(mb, redm[w]);
      best = wthr[w] > best ? wthr[w] : best;
      listed += wlen[w];
    }
    const double sw = wave_sum(s * rescale((double)m, mb == -INFINITY ? 0.0 : mb, tab));
    const int aw = wave_sum(above);
    if (lane() == 0) {
      redd[wave()] = sw;
      redi[wave()] = aw;
    }
    K k[kList / kWave];
    int id[kList / kWave];
    if constexpr (TOP) {
      if (listed > kThreads) {
        // more than a thread each: the waves' first n
        if (len >= a.n) prune(list, len, a.n);
        len = min(len, a.n);
      }
#pragma unroll
      for (int r = 0; r < kList / kWave; ++r) {
        const int i = r * kWave + lane();
        k[r] = i < len ? list.key[i] : 0;
        id[r] = i < len ? list.id[i] : 0;
      }
    }
    wg_barrier();
    double sb = redd[0];
    int ab = redi[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
      sb += redd[w];
      ab += redi[w];
    }
    const PartView<T> pv = part_of<T>(a, row, seg);
    if (a.segs == 1) write_chosen<T>(a, row, chosen, cv, mb, sb, ab);
    int count = 0;
    if constexpr (TOP) {
      // those below `best` are not among the n: at most one entry per thread is left
#pragma unroll
      for (int r = 0; r < kList / kWave; ++r) {
        if (r * kWave >= len) break;
        const bool in = k[r] >= best && k[r] > 0;
        const uint64_t m = __ballot(in);
        int at = 0;
        if (lane() == 0) at = lds_fetch_add(&fill, __popcll(m));
        at = uniform(at) + __popcll(m & ((1ull << lane()) - 1));
        if (in) {
          lkey[at] = k[r];
          lid[at] = id[r];
        }
      }
      wg_barrier();
      count = fill;
      rank_list<K>(lkey, lid, count, [&](int r, K key, int tok) {
        if (r >= a.n) return;
        if (a.segs == 1) {
          write_top<T>(a, row, r, key, tok, mb, sb);
        } else {
          pv.key[r] = key;
          pv.id[r] = tok;
        }
      });
      if (a.segs == 1 && count < a.n) fill_top<T>(a, row, lid, count, mb, sb, redi);
    }
    wg_barrier();  // what lies in LDS is read before the next row writes it
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
  __shared__ int redi[kWaves];
  __shared__ K redk[kWaves];
  __shared__ int fill;
  __shared__ double tabs[kWaves * kWave];
  double* tab = tabs + wave() * kWave;
  init_exp_table_wave(tab);
  for (int row = blockIdx.x; row < a.B; row += gridDim.x) {
    if (threadIdx.x == 0) fill = 0;
    double m = -INFINITY, s = 0.0;
    int above = 0, have = 0;
    K best = 0;
    int chosen = a.ids != nullptr ? a.ids[row] : -1;
    if ((unsigned)chosen >= (unsigned)a.V) chosen = -1;
    const T cv = chosen >= 0 ? static_cast<const T*>(a.x)[(int64_t)row * a.ld + chosen] : (T)0;
    // a thread's first entry, loaded beside the partials
    const int64_t entries = (int64_t)a.segs * a.n;
    K ek = 0;
    int eid = 0, ecount = 0, ej = 0;
    if ((int64_t)threadIdx.x < entries) {
      const PartView<T> pv = part_of<T>(a, row, (int)threadIdx.x / a.n);
      ej = (int)threadIdx.x % a.n;
      ek = pv.key[ej];
      eid = pv.id[ej];
      ecount = pv.part->count;
    }
    // every wave joins all partials for itself: no barrier
    for (int g = lane(); g < a.segs; g += kWave) {
      const PartView<T> pv = part_of<T>(a, row, g);
      const Part p = *pv.part;
      const double mn = fmax(m, p.m), M = mn == -INFINITY ? 0.0 : mn;
      s = s * rescale(m, M, tab) + p.s * rescale(p.m, M, tab);
      m = mn;
      above += p.above;
      have += p.count;
      if (a.n > 0 && p.count == a.n) {
        const K k = pv.key[a.n - 1];
        best = k > best ? k : best;
      }
    }
    const double mb = wave_max(m);
    const double sb = wave_sum(s * rescale(m, mb == -INFINITY ? 0.0 : mb, tab));
    above = wave_sum(above);
    write_chosen<T>(a, row, chosen, cv, mb, sb, above);
    if (a.n == 0) continue;
    have = min(wave_sum(have), a.n);
    best = wave_max(best);
    wg_barrier();  // fill is 0
    if (ej < ecount && ek >= best) {
      const int p = lds_fetch_add(&fill, 1);  // fits: a thread each
      lkey[p] = ek;
      lid[p] = eid;
    }
    for (int64_t e = threadIdx.x + kThreads; e < entries; e += kThreads) {
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
      rank_list<K>(lkey, lid, count, [&](int r, K key, int tok) {
        if (r < a.n) write_top<T>(a, row, r, key, tok, mb, sb);
      });
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

// Segments: as many workgroups as fit the chip at once, two per compute unit, a
// whole chunk or more each (256 x 128256, 20 best, when this was chosen: 49 us, with four 57
// us).  Rows of
// up to three chunks take one: a second launch costs more than the chunks behind one
// another (64 rows of two chunks 10.3 -> 7.8 us, with 20 best 17.8 -> 14.4 us; three:
// 10.4 -> 9.4, 18.2 -> 17.0 us; four: 10.4 -> 10.3, 19.0 -> 19.5 us).
size_t plan_logprobs(LogprobsArgs& a, bool f64, int num_cu, bool one_launch) {
  const int chunk = f64 ? kChunkOf<double> : kChunkOf<float>;
  const int64_t chunks = ((int64_t)a.V + chunk - 1) / chunk, target = 2 * (int64_t)num_cu;
  const int64_t each = one_launch || chunks <= 3 ? chunks : std::min(chunks, (a.B * chunks + target - 1) / target);
  a.seg_chunks = (int)each;
  a.segs = (int)((chunks + each - 1) / each);
  return a.segs == 1 ? 0 : (size_t)a.B * a.segs * (f64 ? part_bytes<double>(a.n) : part_bytes<float>(a.n));
}

hipError_t launch_logprobs(const LogprobsArgs& a, bool f64, hipStream_t s) {
  return f64 ? launch_t<double>(a, s) : launch_t<float>(a, s);
}

}  // namespace plh
