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

// A token's heads, 256 threads: first the sines and cosines of its pairs, then 8
// values of a head at a time (VEC: the turned part is whole runs of 8, halves
// too), or single values.
template <typename T, bool VEC>
__global__ __launch_bounds__(kCacheThreads) void k_rotary(RotaryArgs a) {
  extern __shared__ float2 turn[];
  const int64_t n = blockIdx.x;
  const int64_t pos = a.pairs > 0 ? a.pos[n] : 0;
  for (int i = threadIdx.x; i < a.pairs; i += kCacheThreads) turn[i] = turned(pos, a.freq[i], a.factor);
  wg_barrier();
  const int64_t slot = a.k != nullptr ? a.slots[n] : -1;
  const bool write = slot >= 0 && slot < a.num_slots;
  const int64_t page = write ? slot >> a.page_shift : 0, at = write ? slot & ((1 << a.page_shift) - 1) : 0;
  const int R = 2 * a.pairs, half = a.interleaved ? 0 : a.pairs;
  const int heads = (a.q != nullptr ? a.q_heads : 0) + (write ? 2 * a.kv_heads : 0);
  const int q_heads = a.q != nullptr ? a.q_heads : 0;
  // places of a head where work starts: the first members of the pairs, then the rest
  const int step = VEC ? 8 : 1;
  const int turns = a.interleaved ? R / (VEC ? 8 : 2) : a.pairs / step;
  const int units = turns + (a.D - R) / step;
  for (int u = threadIdx.x; u < heads * units; u += kCacheThreads) {
    const int head = u / units, i = u % units;
    const T* x;
    T* y;
    bool rot = true;
    if (head < q_heads) {
      x = reinterpret_cast<const T*>(a.q) + n * a.ldq + (int64_t)head * a.D;
      y = reinterpret_cast<T*>(a.q_out) + n * a.ldqo + (int64_t)head * a.D;
    } else {
      const int h = head - q_heads;
      rot = h < a.kv_heads;
      const int kvh = rot ? h : h - a.kv_heads;
      x = rot ? reinterpret_cast<const T*>(a.k) + n * a.ldk + (int64_t)kvh * a.D
              : reinterpret_cast<const T*>(a.v) + n * a.ldv + (int64_t)kvh * a.D;
      y = reinterpret_cast<T*>(rot ? a.k_pages : a.v_pages) +
          (((page * a.kv_heads + kvh) << a.page_shift) + at) * a.D;
    }
    const int d = i < turns ? i * (a.interleaved && !VEC ? 2 : step) : R + (i - turns) * step;
    if constexpr (VEC) {
      const Run8<T> p = *reinterpret_cast<const Run8<T>*>(x + d);
      if (i >= turns) {
        *reinterpret_cast<Run8<T>*>(y + d) = p;
      } else if (a.interleaved) {
        Run8<T> o = p;
        if (rot) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 cs = turn[d / 2 + j];
            const float p0 = (float)p.e[2 * j], p1 = (float)p.e[2 * j + 1];
            o.e[2 * j] = (T)(p0 * cs.x - p1 * cs.y);
            o.e[2 * j + 1] = (T)(p1 * cs.x + p0 * cs.y);
          }
        }
        *reinterpret_cast<Run8<T>*>(y + d) = o;
      } else {
        const Run8<T> r = *reinterpret_cast<const Run8<T>*>(x + d + half);
        Run8<T> o = p, z = r;
        if (rot) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float2 cs = turn[d + j];
            const float p0 = (float)p.e[j], p1 = (float)r.e[j];
            o.e[j] = (T)(p0 * cs.x - p1 * cs.y);
            z.e[j] = (T)(p1 * cs.x + p0 * cs.y);
          }
        }
        *reinterpret_cast<Run8<T>*>(y + d) = o;
        *reinterpret_cast<Run8<T>*>(y + d + half) = z;
      }
    } else {
      if (i >= turns) {
        y[d] = x[d];
      } else {
        const int e = a.interleaved ? d + 1 : d + half;
        const T t0 = x[d], t1 = x[e];
        if (rot) {
          const float2 cs = turn[a.interleaved ? d / 2 : d];
          const float p0 = (float)t0, p1 = (float)t1;
          y[d] = (T)(p0 * cs.x - p1 * cs.y);
          y[e] = (T)(p1 * cs.x + p0 * cs.y);
        } else {
          y[d] = t0;
          y[e] = t1;
        }
      }
    }
  }
}

// 16 KB of one page of one layer, four 16-byte loads a thread.
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
// it is read: eight loads, then their eight stores.
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
  if (vec) hipLaunchKernelGGL((k_rotary<T, true>), dim3((unsigned)a.N), dim3(kCacheThreads), lds, s, a);
  else hipLaunchKernelGGL((k_rotary<T, false>), dim3((unsigned)a.N), dim3(kCacheThreads), lds, s, a);
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
