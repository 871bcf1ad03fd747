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
// earlier tests, so nothing but these is kept: every rejection is one pass over the
// node's two rows, which also leaves the sums of its pieces of 512 tokens for the
// draw.  Rows that hold no rejection are touched at their children's tokens alone.
//
// One workgroup a sequence.  Bound by one CU's reads of a node's rows, once a rejection.
#include "plh_kernels.h"
#include "plh_pieces.h"

namespace plh {

namespace {

constexpr int kTreePieces = kTreeV / kPiece;

// The tests that a node's children have failed: their scalars and tokens.
struct Failed {
  const double* iw;   // [m] 1 / W_j
  const double* iz;   // [m] 1 / Z_j
  const int* token;   // [m]
  int m;
  bool replacement, point;  // point: the draft's distribution is its child (q null)
};

__device__ __forceinline__ double positive(double v) { return v > 0.0 ? v : 0.0; }

// r_m of token v, which may be one of the rejected; *s: its share of the draft's distribution then.
__device__ __forceinline__ double left_at(const Failed& f, int v, double p, double q, double* s) {
  double r = p;
  for (int j = 0; j < f.m; ++j) {
    const bool hit = f.token[j] == v;
    r = positive(r * f.iw[j] - (f.point ? (hit ? 1.0 : 0.0) : q * f.iz[j]));
    if (hit && !f.replacement && !f.point) q = 0.0;
  }
  *s = q;
  return positive(r);
}

template <typename TIn>
using PieceRegs = typename PieceGeo<TIn>::V[PieceGeo<TIn>::kLoads];

// The weights r_m of piece s, as load_piece lays them out, and the lane's sum of
// the draft's distribution.
template <typename TIn>
__device__ __forceinline__ double piece_weights(const Failed& f, int s, const PieceRegs<TIn>& x, const PieceRegs<TIn>& y,
                                                double (&w)[PieceGeo<TIn>::kLoads][PieceGeo<TIn>::kVW]) {
  using G = PieceGeo<TIn>;
  bool hit = false;  // a rejected token lies in the piece
  for (int j = 0; j < f.m; ++j) hit |= f.token[j] / kPiece == s;
  double z = 0.0;
#pragma unroll
  for (int j = 0; j < G::kLoads; ++j)
#pragma unroll
    for (int e = 0; e < G::kVW; ++e) {
      w[j][e] = positive((double)x[j][e]);
      z += f.point ? 0.0 : (double)y[j][e];
    }
  if (!hit) {
    for (int i = 0; i < f.m; ++i) {
      const double iw = f.iw[i], iz = f.point ? 0.0 : f.iz[i];
#pragma unroll
      for (int j = 0; j < G::kLoads; ++j)
#pragma unroll
        for (int e = 0; e < G::kVW; ++e) w[j][e] = positive(w[j][e] * iw - (f.point ? 0.0 : (double)y[j][e] * iz));
    }
    return z;
  }
  z = 0.0;
#pragma unroll
  for (int j = 0; j < G::kLoads; ++j)
#pragma unroll
    for (int e = 0; e < G::kVW; ++e) {
      double q = f.point ? 0.0 : (double)y[j][e];
      w[j][e] = left_at(f, s * kPiece + (j * kWave + lane()) * G::kVW + e, (double)x[j][e], q, &q);
      z += q;
    }
  return z;
}

// One pass over a node's rows: the pieces' sums of r_m into `sums`, and the
// calling wave's share of the sum of the draft's distribution.
template <typename TIn, bool WITHQ>
__device__ __forceinline__ double tree_pass(const Failed& f, const TIn* p, const TIn* q, int V, double* sums) {
  using G = PieceGeo<TIn>;
  constexpr int U = 2;  // pieces in flight
  const int n = (V - 1) / kPiece + 1, w = uniform(wave());
  double z = 0.0;
  for (int s = w * U; s < n; s += kWaves * U) {
    PieceRegs<TIn> x[U], y[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      load_piece(p, V, min(s + i, n - 1), x[i]);
      if constexpr (WITHQ) load_piece(q, V, min(s + i, n - 1), y[i]);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (s + i >= n) break;
      double wt[G::kLoads][G::kVW], t = 0.0;
      const double zi = piece_weights<TIn>(f, s + i, x[i], WITHQ ? y[i] : x[i], wt);
      if constexpr (WITHQ) z += zi;
#pragma unroll
      for (int j = 0; j < G::kLoads; ++j)
#pragma unroll
        for (int e = 0; e < G::kVW; ++e) t += wt[j][e];
      t = wave_sum(t);
      if (lane() == 0) sums[s + i] = t;
    }
  }
  return wave_sum(z);
}

template <typename TIn>
__global__ __launch_bounds__(kThreads) void k_verify_tree(TreeArgs a) {
  using G = PieceGeo<TIn>;
  __shared__ double sums[kTreePieces], pv[kTreeNodes], qv[kTreeNodes], us[kTreeNodes], iw[kTreeNodes], iz[kTreeNodes];
  __shared__ double red[kWaves];
  __shared__ int tok[kTreeNodes], par[kTreeNodes], rej[kTreeNodes], path[kTreeNodes];
  const int b = blockIdx.x, V = a.V, pieces = (V - 1) / kPiece + 1;
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
      tok[i] = x;
      par[i] = tested ? up : -1;
      us[i] = a.u[(int64_t)b * a.ldu + i];
      const bool ok = tested && x >= 0 && x < V;
      pv[i] = ok ? (double)row(a.p, up)[x] : 0.0;
      qv[i] = ok && !point ? (double)row(a.q, up)[x] : 1.0;
    }
  }
  wg_barrier();
  // every wave walks on its own, from the same values in the same order
  int cur = 0, i = 0, n = 0, tests = 0;
  bool bad = !sound, empty = false;
  double W = 1.0, w_now = 1.0, z_now = 1.0;  // the node's W, 1 / W and 1 / Z
  Failed f{iw, iz, rej, 0, a.replacement != 0, point};
  if (threadIdx.x == 0 && sound) path[0] = 0;
  while (!bad) {
    int next = INT_MAX;  // the node's next child
    for (int base = (i + 1) / kWave * kWave; base < T; base += kWave) {
      const int j = base + lane();
      const uint64_t m = __ballot(j > i && j < T && par[min(j, kTreeNodes - 1)] == cur);
      if (m != 0) {
        next = base + __builtin_ctzll(m);
        break;
      }
    }
    if (next == INT_MAX) break;
    i = uniform(next);
    const int x = uniform(tok[i]);
    if (x < 0 || x >= V) {
      bad = true;
      break;
    }
    double q = qv[i];
    const double r = left_at(f, x, pv[i], q, &q);
    // p / q as the chain's test has it (NaN accepts); after a rejection a token of
    // which nothing is left is never accepted
    const double ratio = f.m == 0 ? r / q : r > 0.0 ? (r * w_now) / (q * z_now) : 0.0;
    const bool accept = us[tests] < (ratio < 1.0 ? ratio : 1.0);
    ++tests;
    if (accept) {
      cur = i;
      ++n;
      if (threadIdx.x == 0) path[n] = i;
      f.m = 0;
      W = w_now = z_now = 1.0;
      continue;
    }
    wg_barrier();  // all waves have read the scalars of the tests before
    if (threadIdx.x == 0) {
      iw[f.m] = w_now;
      iz[f.m] = z_now;
      rej[f.m] = x;
    }
    ++f.m;
    wg_barrier();
    const double z = point ? tree_pass<TIn, false>(f, row(a.p, cur), nullptr, V, sums)
                           : tree_pass<TIn, true>(f, row(a.p, cur), row(a.q, cur), V, sums);
    if (lane() == 0) red[wave()] = z;
    wg_barrier();
    W = pieces_total([&](int j) { return j < pieces ? sums[j] : 0.0; }, pieces);
    if (!(W > 0.0)) {  // speculative.py:57: nothing is left: the target's row itself
      empty = true;
      break;
    }
    w_now = 1.0 / W;
    if (!f.replacement && !point) {
      double t = red[0];
#pragma unroll
      for (int k = 1; k < kWaves; ++k) t += red[k];
      z_now = 1.0 / t;
    }
  }
  if (bad) {
    for (int j = threadIdx.x; j < a.max_nodes; j += kThreads) out_tok[j] = out_path[j] = -1;
    if (threadIdx.x == 0) {
      a.out_n_acc[b] = -1;
      a.out_n_used[b] = 0;
    }
    return;
  }
  if (empty || f.m == 0) {  // no rejection at the last node: its target row
    f.m = 0;
    wg_barrier();
    (void)tree_pass<TIn, false>(f, row(a.p, cur), nullptr, V, sums);
    wg_barrier();
    W = pieces_total([&](int j) { return j < pieces ? sums[j] : 0.0; }, pieces);
  }
  wg_barrier();  // path
  for (int j = threadIdx.x; j < a.max_nodes; j += kThreads) {
    out_path[j] = j <= n ? path[j] : -1;
    if (j != n) out_tok[j] = j < n ? tok[path[j + 1]] : -1;
  }
  if (wave() != 0) return;
  int t = V - 1;  // sampling.py:98: no mass takes the last id
  if (W > 0.0) {
    const double target = us[tests] * W;
    const Crossing c = cross_pieces([&](int j) { return j < pieces ? sums[j] : 0.0; }, pieces, target);
    if (c.piece >= 0) {
      PieceRegs<TIn> x, y;
      load_piece(row(a.p, cur), V, c.piece, x);
      if (f.m > 0 && !point) load_piece(row(a.q, cur), V, c.piece, y);
      else
#pragma unroll
        for (int j = 0; j < G::kLoads; ++j) y[j] = x[j];
      double w[G::kLoads][G::kVW];
      (void)piece_weights<TIn>(f, c.piece, x, y, w);
      const int hit = pick_in_piece<TIn>(c, target, w);
      if (hit >= 0) t = hit;
    }
  }
  if (lane() == 0) {
    out_tok[n] = t;
    a.out_n_acc[b] = n;
    a.out_n_used[b] = tests + 1;
  }
}

}  // namespace

hipError_t launch_verify_tree(const TreeArgs& a, bool f64, hipStream_t s) {
  if (f64) hipLaunchKernelGGL(k_verify_tree<double>, dim3(a.B), dim3(kThreads), 0, s, a);
  else hipLaunchKernelGGL(k_verify_tree<float>, dim3(a.B), dim3(kThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace plh
