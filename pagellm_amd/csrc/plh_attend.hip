// gfx950 kernels for attention of tree nodes over a paged cache (plh_tree_attention):
// for node i of sequence b and head h, over the keys j that the node sees,
//   o = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale * q . k_j)
// The queries of a sequence that share a key head (its nodes times the group of
// query heads) are rows of one product: keys are the matrix instruction's rows
// and queries its columns, so a lane holds scores of one query, its maximum and
// sum are the lane's own, and the weights are the next product's operand as they
// stand in the registers (a sum may take its keys in any order that both operands
// share).  Keys and values go from HBM to registers in whole rows; nothing of the
// loop passes through LDS.
//
//   k_attend        (chunk of keys, sequence, key head, block of rows): running
//                   maximum and sum, four waves that take blocks of keys in turn,
//                   joined through LDS
//   k_attend_join   (row): the chunks' partial results joined, where there are
//                   several
//
// Values are the rows of the second product.  The matrix instruction wants eight
// keys of one column in a lane; a lane loads 8 columns of 8 keys and pairs their
// halves in registers (v_perm), so that it feeds the instruction for column d = 8 n + j
// with lane n: the order of columns is free too.
#include "plh_device.h"
#include "plh_kernels.h"

#include "pagellm_hip.h"

#include <algorithm>

namespace plh {

namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kAttThreads = 256;
constexpr int kAttWaves = kAttThreads / kWave;
// A wave's own LDS traffic in order (a wave's LDS operations are).
__device__ __forceinline__ void wave_lds_fence() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Waves a SIMD that the registers of a kernel are cut for: what a lane keeps of
// queries, sums, keys and values.
constexpr int attend_waves(int es, int dp, int qt) {
  const int tile = dp * 16 * es / 4 / 64;  // registers of a tile of 16
  const int regs = qt * (tile + dp / 4) + (es == 4 ? 1 : 2) * 2 * tile + 44 + 12 * qt;
  return regs <= 128 ? 4 : regs <= 160 ? 3 : regs <= 256 ? 2 : 1;
}
constexpr int kMostKeys = 1 << 30;
constexpr float kGrow = 8.0f;    // weights stay below 2^8 of the maximum that they are scaled by

// What a lane holds of a tile of 16 keys or queries and of a tile's values, and
// the two products, for 16-bit types.  DP: the head's size, padded.
template <typename T, int DP>
struct Geo {
  static constexpr int kTiles = 2;                   // of 16 keys in a block: the second product's sum
  static constexpr int kSteps = DP / 32;             // 16-byte pieces of a row, a lane
  static constexpr int kE = DP >= 128 ? 8 : DP / 16; // columns of a value row in one load of a lane
  static constexpr int kH = DP / (16 * kE);          // loads of a value row, a lane
  typedef u32x4 Piece;
  typedef uint32_t V __attribute__((ext_vector_type(kE / 2)));
  static __device__ __forceinline__ int piece_at(int s, int g) { return s * 32 + g * 8; }
};

template <int DP>
struct Geo<float, DP> {
  static constexpr int kTiles = 1;
  static constexpr int kSteps = DP / 16;
  static constexpr int kE = 4;
  static constexpr int kH = DP / 64;
  typedef f32x4 Piece;
  typedef f32x4 V;
  static __device__ __forceinline__ int piece_at(int s, int g) { return s * 16 + g * 4; }
};

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

template <typename T>
struct Vec8 {
  typedef bf16x8 type;
};
template <>
struct Vec8<_Float16> {
  typedef f16x8 type;
};

// acc + (a piece of 16 keys) x (that of 16 queries)
template <typename T>
__device__ __forceinline__ f32x4 dot(u32x4 k, u32x4 q, f32x4 acc) {
  typedef typename Vec8<T>::type V;
  return mfma(__builtin_bit_cast(V, k), __builtin_bit_cast(V, q), acc);
}
template <typename T>
__device__ __forceinline__ f32x4 dot(f32x4 k, f32x4 q, f32x4 acc) {
#pragma unroll
  for (int c = 0; c < 4; ++c) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(k[c], q[c], acc, 0, 0, 0);
  return acc;
}

// Two weights as the value product's operand: rounded to the cache's type
// (2^-9 or 2^-12 of a weight, one rounding among those of a sum of many), the
// nearest, so that they lean to no side.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const f32x2 v{a, b};
  if constexpr (__is_same(T, _Float16)) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}

// The largest of the lanes l, l ^ 16, l ^ 32, l ^ 48 (those that share a query), in all of them; and the sum.
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// Whether a loaded vector of values holds an infinity or NaN, and the vector with zeros in their place.
template <typename T, typename V>
__device__ __forceinline__ bool take_finite(V& v) {
  bool bad = false;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool b = !(fabsf(v[i]) < INFINITY);
      bad |= b;
      v[i] = b ? 0.0f : v[i];
    }
  } else {
    constexpr uint32_t e = __is_same(T, _Float16) ? 0x7c00u : 0x7f80u;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(V) / 4); ++i) {
      const bool lo = (v[i] & e) == e, hi = (v[i] & (e << 16)) == (e << 16);
      bad |= lo | hi;
      v[i] = v[i] & (lo ? 0xffff0000u : ~0u) & (hi ? 0x0000ffffu : ~0u);
    }
  }
  return bad;
}

// The running state of QT tiles of 16 rows, one row a column of the products: a
// lane holds row lane % 16 of each, its output columns 4 (lane / 16) + y of a tile.
template <typename T, int DP, int QT>
struct State {
  using G = Geo<T, DP>;
  typename G::Piece q[QT][G::kSteps];
  f32x4 o[QT][G::kH][G::kE];
  float m[QT], l[QT];  // l: over the lane's own keys
  uint64_t bits[QT];   // nodes that the row sees
  int last[QT];        // chains: the last key that it sees
};

template <typename T, int DP, bool FULL>
__device__ __forceinline__ void load_keys(const T* base, int D, typename Geo<T, DP>::Piece (&k)[Geo<T, DP>::kSteps]) {
  using G = Geo<T, DP>;
  const int n = lane() & 15, g = lane() >> 4;
  const T* row = base + n * (FULL ? DP : D);
#pragma unroll
  for (int s = 0; s < G::kSteps; ++s) {
    const int d = G::piece_at(s, g);
    if (FULL || d < D) k[s] = *reinterpret_cast<const typename G::Piece*>(row + d);
    else k[s] = typename G::Piece{};
  }
}

// The lane's four keys (4 g + r) of a tile.
template <typename T, int DP, bool FULL>
__device__ __forceinline__ void load_values(const T* base, int D, typename Geo<T, DP>::V (&v)[4][Geo<T, DP>::kH]) {
  using G = Geo<T, DP>;
  const int n = lane() & 15, g = lane() >> 4;
  const T* row = base + g * 4 * (FULL ? DP : D) + n * G::kE;
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int h = 0; h < G::kH; ++h) {
      const int at = h * 16 * G::kE;
      if (FULL || at + n * G::kE < D) v[r][h] = *reinterpret_cast<const typename G::V*>(row + r * (FULL ? DP : D) + at);
      else v[r][h] = typename G::V{};
    }
}

// A block of a wave: its tiles' places in the pools.  A tile without a page, or
// past the end, is read at the pool's start and masked.
template <int NT>
struct Block {
  int key;
  bool there[NT];
  size_t at[NT];
};

// Four columns of a finished row; a row that sees no key is 0.
template <typename T>
__device__ __forceinline__ void attend_out(const AttendArgs& a, int64_t row, int n, int head, int d, float m, float l,
                                           f32x4 o) {
  typedef T T4 __attribute__((ext_vector_type(4))) __attribute__((aligned(sizeof(T))));
  const float f = l == 0.0f ? 0.0f : 1.0f / l;
  T4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (T)(l == 0.0f ? 0.0f : o[i] * f);
  *reinterpret_cast<T4*>(reinterpret_cast<T*>(a.out) + (int64_t)n * a.ldo + (int64_t)head * a.D + d) = v;
  if (a.lse != nullptr && d == 0) a.lse[row] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.693147180559945309f;
}

// Rows of a sequence and key head: row = node * group + place in the group.
template <typename T, int DP, int QT, bool FULL>
__global__ __launch_bounds__(kAttThreads, attend_waves(sizeof(T), DP, QT)) void k_attend(AttendArgs a) {
  using G = Geo<T, DP>;
  constexpr int NT = G::kTiles, kKeys = 16 * NT;
  constexpr int kRows = 16 * QT, kLd = DP + 4;
  __shared__ __align__(16) float sm_o[kAttWaves][kRows][kLd];
  __shared__ float sm_m[kAttWaves][kRows], sm_l[kAttWaves][kRows];
  const int w = uniform(wave()), n = lane() & 15, g = lane() >> 4;
  // blocks of rows of one unit lie 8 apart: on one XCD, whose L2 then holds the unit's keys
  const int rb = (int)(blockIdx.x / 8 % (unsigned)a.row_blocks);
  const int64_t unit = (int64_t)(blockIdx.x / (8u * (unsigned)a.row_blocks)) * 8 + blockIdx.x % 8;
  if (unit >= (int64_t)a.chunks * a.B * a.kv_heads) return;
  const int kvh = (int)(unit % a.kv_heads), b = (int)(unit / a.kv_heads % a.B), c = (int)(unit / a.kv_heads / a.B);
  const int start = max(a.node_off[b], 0);
  const int nodes = min(min(a.node_off[b + 1], a.N) - start, a.max_nodes);
  const int r0 = rb * kRows;
  if (r0 >= nodes * a.group) return;
  const int ps = 1 << a.page_shift, D = FULL ? DP : a.D;
  const int len = min(max(a.lens[b], 0), kMostKeys);
  // 64 bits: a table's pages may hold more than an int counts
  const int seq_end = (int)min((int64_t)len + nodes, (int64_t)a.ldt << a.page_shift);
  // the last chunk takes what is left where max_len was too small
  const int64_t from64 = (int64_t)c * a.chunk;
  if (c > 0 && from64 >= seq_end) return;
  // this block's rows: keys that all of them see, and the last one that some do
  const int node0 = r0 / a.group, node1 = min((r0 + kRows - 1) / a.group, nodes - 1);
  const int end = min(a.visible == nullptr ? len + node1 + 1 : len + nodes, seq_end);
  const int all = min(a.visible == nullptr ? len + node0 + 1 : len, seq_end);
  const int from = (int)from64, to = c + 1 == a.chunks ? end : (int)min(from64 + a.chunk, (int64_t)end);

  State<T, DP, QT> st;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = r0 + 16 * t + n, node = r / a.group;
    const bool in = node < nodes;
    const T* row = reinterpret_cast<const T*>(a.q) + (int64_t)(start + node) * a.ldq + (int64_t)(kvh * a.group + r % a.group) * D;
#pragma unroll
    for (int s = 0; s < G::kSteps; ++s) {
      const int d = G::piece_at(s, g);
      st.q[t][s] = typename G::Piece{};
      if (in && (FULL || d < D)) {
        typedef typename G::Piece __attribute__((aligned(sizeof(T)))) Loose;
        st.q[t][s] = *reinterpret_cast<const Loose*>(row + d);
      }
    }
    st.bits[t] = a.visible != nullptr && in ? a.visible[start + node] : 0;
    if (nodes < 64) st.bits[t] &= (1ull << nodes) - 1;
    st.last[t] = in ? len + node : -1;
    st.m[t] = -INFINITY;
    st.l[t] = 0.0f;
#pragma unroll
    for (int h = 0; h < G::kH; ++h)
#pragma unroll
      for (int e = 0; e < G::kE; ++e) st.o[t][h][e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // the table through the scalar cache: vector loads return in order, and would
  // wait for the keys in flight
  typedef const __attribute__((address_space(4))) int32_t* Table;
  const Table table = (Table)(a.table + (int64_t)b * a.ldt);
  auto block_at = [&](int key) {
    Block<NT> blk;
    blk.key = key;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int first = key + 16 * t;
      const int page = first < to ? table[first >> a.page_shift] : -1;
      blk.there[t] = (unsigned)page < (unsigned)a.num_pages;
      blk.at[t] = (((size_t)(blk.there[t] ? page : 0) * a.kv_heads + kvh) * ps + (first & (ps - 1))) * D;
    }
    return blk;
  };
  typename G::Piece k[NT][G::kSteps];
  typename G::V v[NT][4][G::kH];
  auto fetch_keys = [&](const Block<NT>& blk) {
#pragma unroll
    for (int t = 0; t < NT; ++t) load_keys<T, DP, FULL>(reinterpret_cast<const T*>(a.k) + blk.at[t], D, k[t]);
  };
  auto fetch_values = [&](const Block<NT>& blk) {
#pragma unroll
    for (int t = 0; t < NT; ++t) load_values<T, DP, FULL>(reinterpret_cast<const T*>(a.v) + blk.at[t], D, v[t]);
  };

  int key = from + w * kKeys;
  Block<NT> blk = block_at(key);
  if (key < to) {
    fetch_keys(blk);
    fetch_values(blk);
  }
  for (; key < to; key += kAttWaves * kKeys) {
    const int after = key + kAttWaves * kKeys;
    const Block<NT> next = block_at(after);
    bool whole = key + kKeys <= min(all, to);
#pragma unroll
    for (int t = 0; t < NT; ++t) whole = whole && blk.there[t];
    float p[QT][NT][4];
#pragma unroll
    for (int c = 0; c < QT; ++c)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f32x4 s{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < G::kSteps; ++i) s = dot<T>(k[t][i], st.q[c][i], s);
#pragma unroll
        for (int r = 0; r < 4; ++r) p[c][t][r] = s[r];
      }
    if (after < to) fetch_keys(next);  // the registers are free again
    if (!whole) {
#pragma unroll
      for (int c = 0; c < QT; ++c)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int x = key + 16 * t + 4 * g + r, node = x - len;
            bool see = blk.there[t] && x < to;
            if (a.visible == nullptr) see = see && x <= st.last[c];
            else see = see && (node < 0 || (node < 64 && (st.bits[c] >> (node & 63) & 1) != 0));
            p[c][t][r] = see ? p[c][t][r] : -INFINITY;
          }
    }
#pragma unroll
    for (int c = 0; c < QT; ++c) {
      float top = -INFINITY;
#pragma unroll
      for (int t = 0; t < NT; ++t)
        top = fmaxf(top, fmaxf(fmaxf(p[c][t][0], p[c][t][1]), fmaxf(p[c][t][2], p[c][t][3])));
      top *= a.scale;
      // the maximum that weights are scaled by moves only where a score would pass
      // it by kGrow: float32 sums hold 2^8 as well as 1
      if (__any(top > st.m[c] + kGrow)) {
        const float m = fmaxf(st.m[c], quad_max(top));
        const float f = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(st.m[c] - m);
        st.m[c] = m;
        st.l[c] *= f;
#pragma unroll
        for (int h = 0; h < G::kH; ++h)
#pragma unroll
          for (int e = 0; e < G::kE; ++e) st.o[c][h][e] *= f;
      }
      const float base = st.m[c] == -INFINITY ? 0.0f : st.m[c];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int r = 0; r < 4; ++r) p[c][t][r] = __builtin_amdgcn_exp2f(fmaf(p[c][t][r], a.scale, -base));
        st.l[c] += (p[c][t][0] + p[c][t][1]) + (p[c][t][2] + p[c][t][3]);
      }
    }
    bool odd = false;  // some value is infinite or NaN, which a weight of 0 must not meet
    if (!whole) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool in = blk.there[t] && key + 16 * t + 4 * g + r < to;
#pragma unroll
          for (int h = 0; h < G::kH; ++h) {
            if (!in) v[t][r][h] = typename G::V{};
            odd |= take_finite<T>(v[t][r][h]);
          }
        }
      odd = __any(odd);
    }
#pragma unroll
    for (int c = 0; c < QT; ++c) {
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int h = 0; h < G::kH; ++h)
#pragma unroll
            for (int e = 0; e < G::kE; ++e)
              st.o[c][h][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[0][r][h][e], p[c][0][r], st.o[c][h][e], 0, 0, 0);
      } else {
        const u32x4 x{pack2<T>(p[c][0][0], p[c][0][1]), pack2<T>(p[c][0][2], p[c][0][3]),
                      pack2<T>(p[c][1][0], p[c][1][1]), pack2<T>(p[c][1][2], p[c][1][3])};
#pragma unroll
        for (int h = 0; h < G::kH; ++h)
#pragma unroll
          for (int e = 0; e < G::kE; ++e) {
            auto pair = [&](int t, int r) {
              return __builtin_amdgcn_perm(v[t][r + 1][h][e / 2], v[t][r][h][e / 2], e & 1 ? 0x07060302u : 0x05040100u);
            };
            st.o[c][h][e] = dot<T>(u32x4{pair(0, 0), pair(0, 2), pair(1, 0), pair(1, 2)}, x, st.o[c][h][e]);
          }
      }
    }
    if (odd) {
      // rare: the infinities and NaN, for the rows that see their keys.  The
      // weights go through the wave's own part of LDS (-1: not seen)
      float* mine = &sm_o[w][0][0];
      static_assert(16 * kKeys <= kRows * kLd, "a wave's weights fit its part");
#pragma unroll
      for (int c = 0; c < QT; ++c) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int x = key + 16 * t + 4 * g + r, node = x - len;
            bool see = blk.there[t] && x < to;
            if (a.visible == nullptr) see = see && x <= st.last[c];
            else see = see && (node < 0 || (node < 64 && (st.bits[c] >> (node & 63) & 1) != 0));
            mine[n * kKeys + 16 * t + 4 * g + r] = see ? p[c][t][r] : -1.0f;
          }
        wave_lds_fence();
#pragma unroll 1
        for (int i = 0; i < kKeys && key + i < to; ++i) {
          const float wt = mine[n * kKeys + i];
          const bool there = i < 16 ? blk.there[0] : blk.there[NT - 1];
          if (!there) continue;
          const T* row = reinterpret_cast<const T*>(a.v) + (i < 16 ? blk.at[0] : blk.at[NT - 1]) + (size_t)(i & 15) * D;
#pragma unroll
          for (int h = 0; h < G::kH; ++h)
#pragma unroll
            for (int y = 0; y < 4; ++y)
#pragma unroll
              for (int e = 0; e < G::kE; ++e) {
                const int d = h * 16 * G::kE + (4 * g + y) * G::kE + e;
                const float x = FULL || d < D ? (float)row[d] : 0.0f;
                if (!(wt < 0.0f) && !(fabsf(x) < INFINITY)) st.o[c][h][e][y] += wt * x;
              }
        }
        wave_lds_fence();
      }
    }
    if (after < to) fetch_values(next);
    blk = next;
  }

#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const float l = quad_sum(st.l[t]);
    if (g == 0) {
      sm_m[w][16 * t + n] = st.m[t];
      sm_l[w][16 * t + n] = l;
    }
#pragma unroll
    for (int h = 0; h < G::kH; ++h)
#pragma unroll
      for (int y = 0; y < 4; ++y)
#pragma unroll
        for (int e = 0; e < G::kE; ++e)
          sm_o[w][16 * t + n][h * 16 * G::kE + (4 * g + y) * G::kE + e] = st.o[t][h][e][y];
  }
  wg_barrier();
  for (int i = threadIdx.x; i < kRows * (DP / 4); i += kAttThreads) {
    const int row = i / (DP / 4), d = i % (DP / 4) * 4, r = r0 + row, node = r / a.group;
    if (node >= nodes || d >= D) continue;
    float m = sm_m[0][row];
#pragma unroll
    for (int x = 1; x < kAttWaves; ++x) m = fmaxf(m, sm_m[x][row]);
    float l = 0.0f;
    f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int x = 0; x < kAttWaves; ++x) {
      const float mx = sm_m[x][row], f = mx == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mx - m);
      const f32x4 ox = *reinterpret_cast<const f32x4*>(&sm_o[x][row][d]);
      // a wave that saw no key is passed over; one whose maximum is infinite brings its NaN along
      if (mx != -INFINITY || sm_l[x][row] != 0.0f) {
        l += f * sm_l[x][row];
        o += f * ox;
      }
    }
    const int head = kvh * a.group + r % a.group;
    const int64_t at = (int64_t)(start + node) * a.heads + head;
    if (a.chunks == 1) {
      attend_out<T>(a, at, start + node, head, d, m, l, o);
    } else {
      const int64_t part = (int64_t)c * a.N * a.heads + at;
      *reinterpret_cast<f32x4*>(a.part_o + part * D + d) = o;
      if (d == 0) *reinterpret_cast<f32x2*>(a.part_ml + 2 * part) = f32x2{m, l};
    }
  }
}

// The chunks of a row joined, a wave a row.
template <typename T>
__global__ __launch_bounds__(kAttThreads) void k_attend_join(AttendArgs a) {
  const int b = blockIdx.y;
  const int start = max(a.node_off[b], 0);
  const int nodes = min(min(a.node_off[b + 1], a.N) - start, a.max_nodes);
  const int64_t i = (int64_t)blockIdx.x * kAttWaves + wave();
  if (i >= (int64_t)nodes * a.heads) return;
  const int64_t end = min((int64_t)min(max(a.lens[b], 0), kMostKeys) + nodes, (int64_t)a.ldt << a.page_shift);
  const int chunks = (int)min((int64_t)a.chunks, max((int64_t)1, (end + a.chunk - 1) / a.chunk));
  const int64_t row = (int64_t)start * a.heads + i, rows = (int64_t)a.N * a.heads;
  float m = -INFINITY;
  for (int c = lane(); c < chunks; c += kWave) m = fmaxf(m, a.part_ml[2 * (c * rows + row)]);
  m = wave_max(m);
  float l = 0.0f;
  f32x4 o{0.0f, 0.0f, 0.0f, 0.0f};
  const int d = lane() * 4;
  for (int c = 0; c < chunks; ++c) {
    const float mx = a.part_ml[2 * (c * rows + row)], lx = a.part_ml[2 * (c * rows + row) + 1];
    if (mx == -INFINITY && lx == 0.0f) continue;  // nothing was written of it
    const float f = mx == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mx - m);
    l += f * lx;
    if (d < a.D) o += f * *reinterpret_cast<const f32x4*>(a.part_o + (c * rows + row) * a.D + d);
  }
  if (d < a.D) attend_out<T>(a, row, start + (int)(i / a.heads), (int)(i % a.heads), d, m, l, o);
}

constexpr int kChunkKeys = kAttWaves * 32;  // a chunk is whole rounds of its waves

template <typename T, int DP, int QT, bool FULL>
hipError_t launch_attend_t(const AttendArgs& a, hipStream_t s) {
  const int64_t units = (int64_t)a.chunks * a.B * a.kv_heads;
  const dim3 grid((unsigned)((units + 7) / 8 * 8 * a.row_blocks));
  hipLaunchKernelGGL((k_attend<T, DP, QT, FULL>), grid, dim3(kAttThreads), 0, s, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.chunks == 1) return e;
  const dim3 join((unsigned)(((int64_t)a.max_nodes * a.heads + kAttWaves - 1) / kAttWaves), (unsigned)a.B);
  hipLaunchKernelGGL(k_attend_join<T>, join, dim3(kAttThreads), 0, s, a);
  return hipGetLastError();
}

template <typename T, int DP>
hipError_t launch_attend_d(const AttendArgs& a, hipStream_t s) {
  if constexpr (DP < 256)
    if (a.row_tiles == 2)
      return a.D == DP ? launch_attend_t<T, DP, 2, true>(a, s) : launch_attend_t<T, DP, 2, false>(a, s);
  return a.D == DP ? launch_attend_t<T, DP, 1, true>(a, s) : launch_attend_t<T, DP, 1, false>(a, s);
}

template <typename T>
hipError_t launch_attend_of(const AttendArgs& a, hipStream_t s) {
  return a.D <= 64 ? launch_attend_d<T, 64>(a, s) : a.D <= 128 ? launch_attend_d<T, 128>(a, s) : launch_attend_d<T, 256>(a, s);
}

}  // namespace

size_t plan_attend(AttendArgs& a, int dtype, int num_cu) {
  const int64_t rows = (int64_t)a.max_nodes * a.group;
  a.row_tiles = rows > 16 && a.D <= 128 ? 2 : 1;
  a.row_blocks = (int)((rows + 16 * a.row_tiles - 1) / (16 * a.row_tiles));
  const int64_t units = std::max<int64_t>(1, (int64_t)a.B * a.kv_heads * a.row_blocks);
  const int64_t most = (a.max_len + kChunkKeys - 1) / kChunkKeys;  // rounds of the longest sequence
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(most / 2, (8LL * num_cu + units - 1) / units));
  a.chunk = (int)((most + want - 1) / want) * kChunkKeys;
  a.chunks = (int)((most * kChunkKeys + a.chunk - 1) / a.chunk);
  return a.chunks == 1 ? 0 : (size_t)a.chunks * a.N * a.heads * (a.D + 2) * sizeof(float);
}

hipError_t launch_attend(AttendArgs a, int dtype, void* ws, hipStream_t s) {
  a.part_o = static_cast<float*>(ws);
  a.part_ml = a.part_o + (size_t)a.chunks * a.N * a.heads * a.D;
  return dtype == PLH_F32 ? launch_attend_of<float>(a, s)
         : dtype == PLH_BF16 ? launch_attend_of<__bf16>(a, s)
                             : launch_attend_of<_Float16>(a, s);
}

}  // namespace plh
