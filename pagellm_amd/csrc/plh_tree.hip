// gfx950 kernel for the accept/resample step over trees of drafted tokens
// (plh_verify_tree), the chain's rule (src/pagellm/engine/speculative.py:38-60)
// applied to siblings in turn.
//
// A node's children are tested in order; a rejected one takes the draft's
// distribution off the target's, and the next is tested against what is left:
//   r_0 = p, s_0 = q, W_0 = Z_0 = 1
//   test child x_j:  u < min(1, (r_j[x] / W_j) / (s_j[x] / Z_j))
//   r_{j+1} = max(r_j / W_j - s_j / Z_j, 0), W_{j+1} = sum r_{j+1}
//   s_{j+1} = s_j without x_j, Z_{j+1} = sum s_{j+1}      (no replacement)
// A token's r_j follows from its p and q and the scalars W and Z of the node's
// earlier tests.  Rows that hold no rejection are touched at their children's tokens
// alone, which are gathered once, ahead of the walk.
//
//   k_tree_clear    the slots for the segments' sums
//   k_verify_tree   (sequence, segment of 8192 tokens): each workgroup walks the tree
//                   on its own; a rejection is a pass over its segment of the node's
//                   two rows, which stay in registers for the next
//
// Passes depend on each other by two sums, which the workgroups of a sequence
// exchange through slots in memory (relaxed atomics of the device's scope; a value is
// its own flag).  A wait ends: a workgroup that has looked for a sum long enough
// computes it itself, with the same instructions in the same order, so that no
// workgroup ever needs another one to run, and all have the same bits.  One
// workgroup a sequence took 34 us where this takes 25 (64 x 16 nodes x 32 000 float64),
// and 132 where this takes 28 (8 x 32 x 128 256).
#include "plh_kernels.h"
#include "plh_pieces.h"

#include <algorithm>

namespace plh {

namespace {

constexpr int kOwn = 2;                             // pieces of a wave
constexpr int kSegPieces = kOwn * kWaves;           // of a segment
constexpr int kSegTokens = kSegPieces * kPiece;
constexpr int kSegments = kTreeV / kSegTokens;      // at most, of a row: a lane each
static_assert(kSegments <= kWave, "a wave reads the segments' sums");
constexpr int kSharedPasses = 32;                   // of a sequence; later ones are computed by each workgroup alone
constexpr uint64_t kEmpty = ~0ull;                  // a NaN that no sum has

__host__ __device__ constexpr int segments_of(int V) { return (V - 1) / kSegTokens + 1; }

__device__ __forceinline__ double positive(double v) { return v > 0.0 ? v : 0.0; }

// One step of r.  Spelled out, so that every copy of it rounds alike.
__device__ __forceinline__ double less(double r, double iw, double s, double iz) {
  return positive(__builtin_fma(-s, iz, r * iw));
}

// The tests that a node's children have failed: their scalars and tokens.
struct Failed {
  const double* iw;   // [m] 1 / W_j
  const double* iz;   // [m] 1 / Z_j
  const int* token;   // [m]
  int m;
  bool replacement, point;  // point: the draft's distribution is its child (q null)
};

// r_m of token v, which may be one of the rejected, and its s_m.
__device__ __forceinline__ double left_at(const Failed& f, int v, double p, double q, double* s) {
  double r = positive(p);
  for (int j = 0; j < f.m; ++j) {
    const bool hit = f.token[j] == v;
    r = f.point ? less(r, f.iw[j], hit ? 1.0 : 0.0, 1.0) : less(r, f.iw[j], q, f.iz[j]);
    if (hit && !f.replacement && !f.point) q = 0.0;
  }
  *s = q;
  return r;
}

// A piece's r and s, a lane's share.
template <typename TIn>
struct Piece {
  using G = PieceGeo<TIn>;
  double r[G::kLoads][G::kVW];
  typename G::V s[G::kLoads];
};

template <typename TIn>
__device__ __forceinline__ void load_rows(const TIn* p, const TIn* q, int V, int piece, Piece<TIn>& x) {
  using G = PieceGeo<TIn>;
  typename G::V y[G::kLoads];
  load_piece(p, V, piece, y);
  if (q != nullptr) load_piece(q, V, piece, x.s);
#pragma unroll
  for (int j = 0; j < G::kLoads; ++j) {
#pragma unroll
    for (int e = 0; e < G::kVW; ++e) x.r[j][e] = positive((double)y[j][e]);
  }
  if (q == nullptr)
#pragma unroll
    for (int j = 0; j < G::kLoads; ++j)
#pragma unroll
      for (int e = 0; e < G::kVW; ++e) x.s[j][e] = TIn(0);
}

// The piece after failed test j of f.
template <typename TIn>
__device__ __forceinline__ void step_piece(const Failed& f, int j, int piece, Piece<TIn>& x) {
  using G = PieceGeo<TIn>;
  const double iw = f.iw[j], iz = f.iz[j];
  const int token = f.token[j];
#pragma unroll
  for (int l = 0; l < G::kLoads; ++l)
#pragma unroll
    for (int e = 0; e < G::kVW; ++e) x.r[l][e] = less(x.r[l][e], iw, (double)x.s[l][e], iz);
  if (token / kPiece != piece) return;
#pragma unroll
  for (int l = 0; l < G::kLoads; ++l)
#pragma unroll
    for (int e = 0; e < G::kVW; ++e)
      if (piece * kPiece + (l * kWave + lane()) * G::kVW + e == token) {
        // its share of a point draft is all of it, and was taken as 0
        if (f.point) x.r[l][e] = positive(x.r[l][e] - 1.0);
        else if (!f.replacement) x.s[l][e] = TIn(0);
      }
}

// The piece's sums of r and s.
template <typename TIn>
__device__ __forceinline__ void piece_sums(const Piece<TIn>& x, double* r, double* s) {
  using G = PieceGeo<TIn>;
  double a = 0.0, b = 0.0;
#pragma unroll
  for (int l = 0; l < G::kLoads; ++l)
#pragma unroll
    for (int e = 0; e < G::kVW; ++e) {
      a += x.r[l][e];
      b += (double)x.s[l][e];
    }
  *r = wave_sum(a);
  *s = wave_sum(b);
}

struct TreeLds {
  double pv[kTreeNodes], qv[kTreeNodes], us[kTreeNodes], iw[kTreeNodes], iz[kTreeNodes];
  double piece_r[kSegPieces], piece_s[kSegPieces], seg_r[kWave], seg_s[kWave];
  int tok[kTreeNodes], par[kTreeNodes], rej[kTreeNodes], path[kTreeNodes];
  int missing;
};

// The calling workgroup's sums of the pieces in l.piece_r and l.piece_s, in one order.
__device__ __forceinline__ void segment_sums(const TreeLds& l, double* r, double* s) {
  const bool in = lane() < kSegPieces;
  *r = wave_sum(in ? l.piece_r[lane() & (kSegPieces - 1)] : 0.0);
  *s = wave_sum(in ? l.piece_s[lane() & (kSegPieces - 1)] : 0.0);
}

// Sums of r and s of the row's segments into l.seg_r and l.seg_s: this workgroup's,
// whose pieces' stand in l, for the others, theirs from the slots, and what does not
// come from the rows themselves.
template <typename TIn>
__device__ __forceinline__ void exchange(const TreeArgs& a, TreeLds& l, const Failed& f, const TIn* p, const TIn* q, int b,
                                         int seg, int pass) {
  const int n = segments_of(a.V);
  wg_barrier();
  if (n == 1) {
    if (wave() == 0) {
      double r, s;
      segment_sums(l, &r, &s);
      if (lane() == 0) {
        l.seg_r[0] = r;
        l.seg_s[0] = s;
      }
    }
    wg_barrier();
    return;
  }
  const bool shared = pass < kSharedPasses;
  if (wave() == 0) {
    double r, s;
    segment_sums(l, &r, &s);
    unsigned long long* slot =
        a.slots + (((size_t)b * a.passes + (shared ? pass : 0)) * n + (lane() < n ? lane() : 0)) * 2;
    uint64_t x = kEmpty, y = kEmpty;
    if (lane() == seg) {
      // a sum that is NaN is no flag
      x = r == r ? __builtin_bit_cast(uint64_t, r) : 0x7ff8000000000000ull;
      y = s == s ? __builtin_bit_cast(uint64_t, s) : 0x7ff8000000000000ull;
      if (shared) {
        __hip_atomic_store(PLH_GLB(unsigned long long, slot), x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(PLH_GLB(unsigned long long, slot + 1), y, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
    for (int i = 0; shared && i < a.looks; ++i) {
      const bool look = lane() < n && (x == kEmpty || y == kEmpty);
      if (__ballot(look) == 0) break;
      if (look) {
        x = __hip_atomic_load(PLH_GLB(unsigned long long, slot), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        y = __hip_atomic_load(PLH_GLB(unsigned long long, slot + 1), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
    l.seg_r[lane()] = lane() < n ? __builtin_bit_cast(double, x) : 0.0;
    l.seg_s[lane()] = lane() < n ? __builtin_bit_cast(double, y) : 0.0;
    const uint64_t none = __ballot(lane() < n && (x == kEmpty || y == kEmpty));
    if (lane() == 0) l.missing = none != 0 ? __builtin_ctzll(none) : n;
  }
  wg_barrier();
  const double own_r = l.piece_r[lane() & (kSegPieces - 1)], own_s = l.piece_s[lane() & (kSegPieces - 1)];
  int g = uniform(l.missing);
  if (g == n) return;
  for (; g < n; ++g) {
    const uint64_t x = __builtin_bit_cast(uint64_t, l.seg_r[g]), y = __builtin_bit_cast(uint64_t, l.seg_s[g]);
    if (uniform(x) != kEmpty && uniform(y) != kEmpty) continue;
    wg_barrier();
#pragma unroll 1
    for (int k = 0; k < kOwn; ++k) {
      const int piece = g * kSegPieces + wave() * kOwn + k;
      double r = 0.0, s = 0.0;
      if (piece * kPiece < a.V) {
        Piece<TIn> v;
        load_rows(p, q, a.V, piece, v);
        for (int j = 0; j < f.m; ++j) step_piece(f, j, piece, v);
        piece_sums(v, &r, &s);
      }
      if (lane() == 0) {
        l.piece_r[wave() * kOwn + k] = r;
        l.piece_s[wave() * kOwn + k] = s;
      }
    }
    wg_barrier();
    if (wave() == 0) {
      double r, s;
      segment_sums(l, &r, &s);
      if (lane() == 0) {
        l.seg_r[g] = r;
        l.seg_s[g] = s;
      }
    }
    wg_barrier();
  }
  if (wave() == 0 && lane() < kSegPieces) {
    l.piece_r[lane()] = own_r;
    l.piece_s[lane()] = own_s;
  }
  wg_barrier();
}

__global__ __launch_bounds__(kThreads) void k_tree_clear(unsigned long long* slots, size_t n) {
  const size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x;
  if (i < n) slots[i] = kEmpty;
}

template <typename TIn>
// (float64 spills at 128 registers: 64 x 32 000 27.8 against 24.7 us)
__global__ __launch_bounds__(kThreads, sizeof(TIn) == 8 ? 2 : 4) void k_verify_tree(TreeArgs a) {
  using G = PieceGeo<TIn>;
  __shared__ TreeLds l;
  const int segs = segments_of(a.V), b = blockIdx.x / segs, seg = blockIdx.x % segs, V = a.V;
  const int start = a.node_off[b], T = a.node_off[b + 1] - start;
  int32_t* out_tok = a.out_tokens + (size_t)b * a.max_nodes;
  int32_t* out_path = a.out_path + (size_t)b * a.max_nodes;
  const bool point = a.q == nullptr;
  const bool sound = start >= 0 && T > 0 && T <= a.max_nodes && start <= a.N - T;
  auto row = [&](const void* base, int node) { return reinterpret_cast<const TIn*>(base) + (int64_t)(start + node) * a.ld; };
  if (sound) {
    for (int i = threadIdx.x; i < T; i += kThreads) {
      const int x = a.tokens[start + i], up = a.parents[start + i];
      const bool tested = i > 0 && up >= 0 && up < i;
      l.tok[i] = x;
      l.par[i] = tested ? up : -1;
      l.us[i] = a.u[(int64_t)b * a.ldu + i];
      const bool ok = tested && x >= 0 && x < V;
      l.pv[i] = ok ? (double)row(a.p, up)[x] : 0.0;
      l.qv[i] = ok && !point ? (double)row(a.q, up)[x] : 1.0;
    }
  }
  wg_barrier();
  // every wave of every workgroup walks on its own, from the same values in the same order
  int cur = 0, i = 0, n = 0, tests = 0, pass = 0;
  bool bad = !sound;
  double W = 0.0, w_now = 1.0, z_now = 1.0;  // the node's W, 1 / W and 1 / Z
  Failed f{l.iw, l.iz, l.rej, 0, a.replacement != 0, point};
  Piece<TIn> mine[kOwn];
  const int piece0 = seg * kSegPieces + wave() * kOwn;
  // The segment's part of pass f.m of the current node, and the row's sums of it.
  auto sum_up = [&](const TIn* p, const TIn* q) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
      const int piece = piece0 + k;
      double r = 0.0, s = 0.0;
      if (piece * kPiece < V) {
        if (f.m <= 1) load_rows(p, q, V, piece, mine[k]);
        if (f.m > 0) step_piece(f, f.m - 1, piece, mine[k]);
        piece_sums(mine[k], &r, &s);
      }
      if (lane() == 0) {
        l.piece_r[wave() * kOwn + k] = r;
        l.piece_s[wave() * kOwn + k] = s;
      }
    }
    exchange(a, l, f, p, q, b, seg, pass);
    ++pass;
    W = wave_sum(l.seg_r[lane()]);  // past the row's segments: 0
    return wave_sum(l.seg_s[lane()]);
  };
  if (threadIdx.x < kWave) l.seg_r[lane()] = l.seg_s[lane()] = 0.0;
  if (threadIdx.x == 0 && sound) l.path[0] = 0;
  bool last = false;  // the target's row of the last node, for the draw
  while (!bad) {
    if (!last) {
      int next = INT_MAX;  // the node's next child
      for (int base = (i + 1) / kWave * kWave; base < T; base += kWave) {
        const int j = base + lane();
        const uint64_t m = __ballot(j > i && j < T && l.par[min(j, kTreeNodes - 1)] == cur);
        if (m != 0) {
          next = base + __builtin_ctzll(m);
          break;
        }
      }
      last = next == INT_MAX;
      if (last && f.m > 0) break;  // what the rejections left stands in the sums
      if (!last) {
        i = uniform(next);
        const int x = uniform(l.tok[i]);
        if (x < 0 || x >= V) {
          bad = true;
          break;
        }
        double q = l.qv[i];
        const double r = f.m == 0 ? l.pv[i] : left_at(f, x, l.pv[i], q, &q);
        // p / q as the chain's test has it (NaN accepts); after a rejection a token of
        // which nothing is left is never accepted
        const double ratio = f.m == 0 ? r / q : r > 0.0 ? (r * w_now) / (q * z_now) : 0.0;
        const bool accept = l.us[tests] < (ratio < 1.0 ? ratio : 1.0);
        ++tests;
        if (accept) {
          cur = i;
          ++n;
          if (threadIdx.x == 0) l.path[n] = i;
          f.m = 0;
          w_now = z_now = 1.0;
          continue;
        }
        wg_barrier();  // all waves have read the scalars of the tests before
        if (threadIdx.x == 0) {
          l.iw[f.m] = w_now;
          l.iz[f.m] = z_now;
          l.rej[f.m] = x;
        }
        ++f.m;
      }
    }
    if (last) f.m = 0;
    wg_barrier();
    const double z = sum_up(row(a.p, cur), point || last ? nullptr : row(a.q, cur));
    if (last) break;
    // speculative.py:57: nothing is left: the target's row itself
    last = !(W > 0.0);
    w_now = 1.0 / W;
    if (!f.replacement && !point) z_now = 1.0 / z;
  }
  if (bad) {
    if (seg != 0) return;
    for (int j = threadIdx.x; j < a.max_nodes; j += kThreads) out_tok[j] = out_path[j] = -1;
    if (threadIdx.x == 0) {
      a.out_n_acc[b] = -1;
      a.out_n_used[b] = 0;
    }
    return;
  }
  // the segment in which the running total crosses u W draws the token
  const double target = l.us[tests] * W;
  int owner = 0;
  double before = 0.0;
  bool crossed = false;
  if (W > 0.0) {
    const double v = l.seg_r[lane()];
    const double incl = wave_scan_incl(v, 0.0, OpAdd{});
    const uint64_t some = __ballot(v > 0.0), over = __ballot(v > 0.0 && incl > target);
    crossed = over != 0;
    owner = over != 0 ? __builtin_ctzll(over) : some != 0 ? 63 - __builtin_clzll(some) : 0;
    before = lane_value(incl - v, owner);
  }
  owner = uniform(owner);
  if (seg != owner) return;
  for (int j = threadIdx.x; j < a.max_nodes; j += kThreads) {
    out_path[j] = j <= n ? l.path[j] : -1;
    if (j != n) out_tok[j] = j < n ? l.tok[l.path[j + 1]] : -1;
  }
  Crossing c{-1, false, 0.0};
  if (W > 0.0) {
    const double v = lane() < kSegPieces ? l.piece_r[lane() & (kSegPieces - 1)] : 0.0;
    const double incl = before + wave_scan_incl(v, 0.0, OpAdd{});
    const uint64_t some = __ballot(v > 0.0), over = crossed ? __ballot(v > 0.0 && incl > target) : 0;
    if (some != 0) {
      const int k = over != 0 ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
      c = Crossing{k, over != 0, lane_value(incl - v, k)};
    }
  }
  if (wave() != (c.piece < 0 ? 0 : c.piece / kOwn)) return;
  int t = V - 1;  // sampling.py:98: no mass takes the last id
  if (c.piece >= 0) {
    double w[G::kLoads][G::kVW];
#pragma unroll
    for (int j = 0; j < G::kLoads; ++j)
#pragma unroll
      for (int e = 0; e < G::kVW; ++e) {
        double x = mine[0].r[j][e], y = mine[kOwn - 1].r[j][e];
        asm volatile("" : "+v"(x), "+v"(y));  // values: a choice of places would put both pieces into memory
        w[j][e] = c.piece % kOwn == 0 ? x : y;
      }
    c.piece += seg * kSegPieces;
    const int hit = pick_in_piece<TIn>(c, target, w);
    if (hit >= 0) t = hit;
  }
  if (lane() == 0) {
    out_tok[n] = t;
    a.out_n_acc[b] = n;
    a.out_n_used[b] = tests + 1;
  }
}

}  // namespace

size_t tree_ws_bytes(int B, int V, int max_nodes) {
  const size_t n = segments_of(V);
  // a pass a test, and one at the end
  return n == 1 ? 0 : (size_t)B * std::min(max_nodes + 1, kSharedPasses) * n * 2 * sizeof(uint64_t);
}

hipError_t launch_verify_tree(TreeArgs a, bool f64, void* ws, hipStream_t s) {
  const int segs = segments_of(a.V);
  a.slots = static_cast<unsigned long long*>(ws);
  a.passes = std::min(a.max_nodes + 1, kSharedPasses);
  if (segs > 1) {
    const size_t n = tree_ws_bytes(a.B, a.V, a.max_nodes) / sizeof(uint64_t);
    hipLaunchKernelGGL(k_tree_clear, dim3((unsigned)((n + kThreads - 1) / kThreads)), dim3(kThreads), 0, s, a.slots, n);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  const dim3 grid((unsigned)((int64_t)a.B * segs));
  if (f64) hipLaunchKernelGGL(k_verify_tree<double>, grid, dim3(kThreads), 0, s, a);
  else hipLaunchKernelGGL(k_verify_tree<float>, grid, dim3(kThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace plh
