// gfx950 kernels for the pages of a key and value cache:
//   k_rotary   rotary positions of a step's queries and keys, keys and values
//              written into their places (plh_rotary_append)
//   k_copy     pages of all layers copied (plh_copy_pages)
//   k_keep     the accepted nodes' keys and values of all layers moved together
//              (plh_keep_nodes)
// All are bound by the bytes they move, small calls by their launch.
//
// Rotary: pair i of a head is turned by pos * f_i radians and scaled by a factor.
// At position 2^20 a float32 angle is 2^-5 off: the angle is formed in float64 as
// turns, whose whole part is dropped exactly, and only the rest, at most half a
// turn, goes to float32 for its sine and cosine.
#include "plh_device.h"
#include "plh_kernels.h"

#include "pagellm_hip.h"

#include <algorithm>
#include <type_traits>

namespace plh {

namespace {

constexpr int kCacheThreads = 256;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Run8 {
  T e[8];
};

// cos and sin of pos * f radians, times the factor
__device__ __forceinline__ float2 turned(int64_t pos, double f, float factor) {
  double t = (double)pos * (f * 0.15915494309189533577);  // turns
  t -= rint(t);
  float s, c;
  sincospif(2.0f * (float)t, &s, &c);
  return float2{c * factor, s * factor};
}

// What a unit of work holds: 8 values of a head (VEC: the turned part is whole runs
// of 8, halves too) or one, and their pairs' other members, where those lie elsewhere.
template <typename T, bool VEC>
struct TurnUnit {
  typedef std::conditional_t<VEC, Run8<T>, T> Run;
  Run x, z;
  int head, d;  // d: the first value's place
  bool turn;    // of a turned pair
};

// A token's heads, a unit a thread at a time.  Units are asked for two ahead, the
// first ones before the sines and cosines are computed: 8192 tokens of 32 + 8 + 8 heads
// of 128 values of 16 bits 56 -> 44 us, 4.6 TB/s.  A decode step of 64 tokens takes 4.2.
constexpr int kRotaryAhead = 2;

template <typename T, bool VEC>
__global__ __launch_bounds__(kCacheThreads) void k_rotary(RotaryArgs a) {
  extern __shared__ float2 turn[];
  typedef TurnUnit<T, VEC> Unit;
  typedef typename Unit::Run Run;
  const int64_t n = blockIdx.x;
  const int R = 2 * a.pairs, q_heads = a.q != nullptr ? a.q_heads : 0;
  const bool apart = !(VEC && a.interleaved);  // a pair's members are in two runs
  const int other = a.interleaved ? 1 : a.pairs;
  constexpr int kStep = VEC ? 8 : 1;
  const int first_step = a.interleaved && !VEC ? 2 : kStep;
  const int turns = a.interleaved ? R / first_step : a.pairs / kStep, units = turns + (a.D - R) / kStep;
  const int all = (q_heads + (a.k != nullptr ? 2 * a.kv_heads : 0)) * units;
  auto fetch = [&](int u, Unit& w) __attribute__((always_inline)) {
    if (u >= all) return;
    w.head = u / units;
    const int i = u % units, h = w.head - q_heads;
    w.turn = i < turns;
    w.d = w.turn ? i * first_step : R + (i - turns) * kStep;
    const T* x = h < 0            ? reinterpret_cast<const T*>(a.q) + n * a.ldq + (int64_t)w.head * a.D
                 : h < a.kv_heads ? reinterpret_cast<const T*>(a.k) + n * a.ldk + (int64_t)h * a.D
                                  : reinterpret_cast<const T*>(a.v) + n * a.ldv + (int64_t)(h - a.kv_heads) * a.D;
    w.x = *reinterpret_cast<const Run*>(x + w.d);
    if (w.turn && apart) w.z = *reinterpret_cast<const Run*>(x + w.d + other);
  };
  Unit w[kRotaryAhead];
  const int threads = blockDim.x;
  int u = threadIdx.x;
#pragma unroll
  for (int e = 0; e < kRotaryAhead; ++e) fetch(u + e * threads, w[e]);
  const int64_t slot = a.k != nullptr ? a.slots[n] : -1;
  const int64_t pos = a.pairs > 0 ? a.pos[n] : 0;
  for (int i = threadIdx.x; i < a.pairs; i += threads) turn[i] = turned(pos, a.freq[i], a.factor);
  wg_barrier();
  const bool write = slot >= 0 && slot < a.num_slots;
  const int64_t page = write ? slot >> a.page_shift : 0, at = write ? slot & ((1 << a.page_shift) - 1) : 0;
  auto turn_pair = [](T& p, T& q, float2 cs) {
    const float p0 = (float)p, p1 = (float)q;
    p = (T)(p0 * cs.x - p1 * cs.y);
    q = (T)(p1 * cs.x + p0 * cs.y);
  };
  auto finish = [&](Unit& w) __attribute__((always_inline)) {
    const int h = w.head - q_heads;
    if (h >= 0 && !write) return;
    const bool value = h >= a.kv_heads;
    T* y = h < 0 ? reinterpret_cast<T*>(a.q_out) + n * a.ldqo + (int64_t)w.head * a.D
                 : reinterpret_cast<T*>(value ? a.v_pages : a.k_pages) +
                       (((page * a.kv_heads + (value ? h - a.kv_heads : h)) << a.page_shift) + at) * a.D;
    if (w.turn && !value) {
      if constexpr (VEC) {
        if (apart) {
#pragma unroll
          for (int j = 0; j < 8; ++j) turn_pair(w.x.e[j], w.z.e[j], turn[w.d + j]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) turn_pair(w.x.e[2 * j], w.x.e[2 * j + 1], turn[w.d / 2 + j]);
        }
      } else {
        turn_pair(w.x, w.z, turn[a.interleaved ? w.d / 2 : w.d]);
      }
    }
    *reinterpret_cast<Run*>(y + w.d) = w.x;
    if (w.turn && apart) *reinterpret_cast<Run*>(y + w.d + other) = w.z;
  };
  for (; u < all; u += kRotaryAhead * threads) {
#pragma unroll
    for (int e = 0; e < kRotaryAhead; ++e)
      if (u + e * threads < all) finish(w[e]);
    // the next ones, if any
#pragma unroll
    for (int e = 0; e < kRotaryAhead; ++e) fetch(u + (kRotaryAhead + e) * threads, w[e]);
  }
}

// 16 KB of one page of one layer, four 16-byte loads a thread: 512 pairs of 32 KB in
// 16 layers, keys and values, 204 us, 5.3 TB/s (a large copy's rate); 8 pairs 4.6 us.
constexpr int kCopyLoads = 4;
constexpr int kCopyBytes = kCopyLoads * kCacheThreads * 16;

__global__ __launch_bounds__(kCacheThreads) void k_copy(CopyArgs a) {
  const int pair = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
  const int src = a.src[pair], dst = a.dst[pair];
  if ((unsigned)src >= (unsigned)a.num_pages || (unsigned)dst >= (unsigned)a.num_pages || src == dst) return;
  char* pool = reinterpret_cast<char*>(blockIdx.z == 0 ? a.k : a.v) + (int64_t)blockIdx.y * a.layer_bytes;
  const char* from = pool + (int64_t)src * a.page_bytes;
  char* to = pool + (int64_t)dst * a.page_bytes;
  const int64_t at = (int64_t)slice * kCopyBytes + threadIdx.x * 16;
  u32x4 x[kCopyLoads];
#pragma unroll
  for (int i = 0; i < kCopyLoads; ++i) {
    const int64_t o = at + i * kCacheThreads * 16;
    if (o < a.page_bytes) x[i] = *reinterpret_cast<const u32x4*>(from + o);
  }
#pragma unroll
  for (int i = 0; i < kCopyLoads; ++i) {
    const int64_t o = at + i * kCacheThreads * 16;
    if (o < a.page_bytes) *reinterpret_cast<u32x4*>(to + o) = x[i];
  }
}

// 16 bytes of a token's row of one layer, pool and head: a thread walks the path.
// Place j takes node path[j] >= j, so a later node's place is never written before
// it is read: eight loads, then their eight stores.  64 sequences x 32 layers, 8 heads
// of 128: 10 us, a launch and two rounds of loads and stores; 8 x 16 layers 4.1 us.
constexpr int kKeepNodes = 64;  // of the path at a time
constexpr int kKeepLoads = 8;

__global__ __launch_bounds__(kCacheThreads) void k_keep(KeepArgs a) {
  __shared__ int64_t from[kKeepNodes], to[kKeepNodes];  // in tokens of a head's rows
  const int b = blockIdx.y;
  const int n = min(a.n_acc[b], a.ldp - 1);
  const int64_t len = max(a.lens[b], 0);
  const int64_t i = (int64_t)blockIdx.x * kCacheThreads + threadIdx.x;
  const int piece = (int)(i % a.pieces), head = (int)(i / a.pieces % a.kv_heads);
  const int64_t at = i / a.pieces / a.kv_heads;
  const bool in = at < 2 * (int64_t)a.layers;
  char* pool = reinterpret_cast<char*>(at & 1 ? a.v : a.k) + (in ? at / 2 : 0) * a.layer_bytes;
  const int64_t row_bytes = (int64_t)a.pieces * 16;
  char* base = pool + ((int64_t)head << a.page_shift) * row_bytes + piece * 16;
  for (int j0 = 1; j0 <= n; j0 += kKeepNodes) {
    const int m = min(n - j0 + 1, kKeepNodes);
    if ((int)threadIdx.x < m) {
      const int j = j0 + threadIdx.x, node = a.path[(int64_t)b * a.ldp + j];
      int64_t place[2] = {len + node, len + j};
      bool ok = node > j;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int64_t p = place[s] >> a.page_shift;
        const int page = ok && p < a.ldt ? a.table[(int64_t)b * a.ldt + p] : -1;
        ok = ok && (unsigned)page < (unsigned)a.num_pages;
        place[s] = (((int64_t)page * a.kv_heads) << a.page_shift) + (place[s] & ((1 << a.page_shift) - 1));
      }
      from[threadIdx.x] = ok ? place[0] : -1;
      to[threadIdx.x] = place[1];
    }
    wg_barrier();
    if (in) {
      for (int j = 0; j < m; j += kKeepLoads) {
        u32x4 x[kKeepLoads];
#pragma unroll
        for (int e = 0; e < kKeepLoads; ++e)
          if (j + e < m && from[j + e] >= 0) x[e] = *reinterpret_cast<const u32x4*>(base + from[j + e] * row_bytes);
#pragma unroll
        for (int e = 0; e < kKeepLoads; ++e)
          if (j + e < m && from[j + e] >= 0) *reinterpret_cast<u32x4*>(base + to[j + e] * row_bytes) = x[e];
      }
    }
    wg_barrier();
  }
}

template <typename T>
hipError_t launch_rotary_t(const RotaryArgs& a, hipStream_t s) {
  const bool vec = a.pairs % (a.interleaved ? 4 : 8) == 0 && a.D % 8 == 0;
  const size_t lds = (size_t)std::max(a.pairs, 1) * sizeof(float2);
  // two units a thread, if that takes no more threads than a workgroup's
  const int64_t heads = (a.q != nullptr ? a.q_heads : 0) + (a.k != nullptr ? 2 * (int64_t)a.kv_heads : 0);
  const int64_t units = heads * (vec ? a.D / 8 - (a.interleaved ? 0 : a.pairs / 8) : a.D - a.pairs);
  const dim3 block((unsigned)std::min<int64_t>(kCacheThreads, std::max<int64_t>(1, (units + 127) / 128) * 64));
  if (vec) hipLaunchKernelGGL((k_rotary<T, true>), dim3((unsigned)a.N), block, lds, s, a);
  else hipLaunchKernelGGL((k_rotary<T, false>), dim3((unsigned)a.N), block, lds, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_rotary(const RotaryArgs& a, int dtype, hipStream_t s) {
  return dtype == PLH_F32 ? launch_rotary_t<float>(a, s)
         : dtype == PLH_BF16 ? launch_rotary_t<__bf16>(a, s)
                             : launch_rotary_t<_Float16>(a, s);
}

hipError_t launch_copy_pages(CopyArgs a, int n, hipStream_t s) {
  a.slices = (int)((a.page_bytes + kCopyBytes - 1) / kCopyBytes);
  hipLaunchKernelGGL(k_copy, dim3((unsigned)((int64_t)n * a.slices), (unsigned)a.layers, 2), dim3(kCacheThreads), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_keep(const KeepArgs& a, int B, hipStream_t s) {
  const int64_t threads = 2 * (int64_t)a.layers * a.kv_heads * a.pieces;
  hipLaunchKernelGGL(k_keep, dim3((unsigned)((threads + kCacheThreads - 1) / kCacheThreads), (unsigned)B),
                     dim3(kCacheThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace plh
