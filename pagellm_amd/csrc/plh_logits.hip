// gfx950 kernel for biases, penalties and grammar masks on a batch's logits
// (plh_process_logits): of row b
//   v = x + bias                    tokens of the bias list
//   v = v > 0 ? v / r : v * r       tokens of the history
//   v = v - (f * n + p)             tokens that occur n > 0 times among the outputs
//   v = -inf                        tokens the mask rules out
// and for the chosen tokens' processed logits (plh_token_logits).
//
// One workgroup per row and chunk of kProcChunk tokens.  The history and the
// bias list are sparse and unsorted, the logits dense: the workgroup counts the
// history's tokens of its chunk in an LDS table (integer atomics: the counts do
// not depend on their order), marks the biased ones in a second one, and then
// walks its chunk once, looking both tables and the mask up by position.  Rows
// whose parameters are neutral skip the tables.  A chunk reads the whole history
// (from L2), 4 H bytes beside the 8 * kProcChunk of its logits.
//
// Bound by the read and write of the logits: 256 x 128 256, half of the rows with
// 2048-token histories and half with masks, 65 us (logits not in the caches; a copy of them
// 50 us), 54 us where they are.  In place, masks that leave most quads alone 34 us.  Chunks of 4096 with at most 64 registers put four
// workgroups on a CU (chunks of 8192, two: 60 us); four history loads in flight a thread
// (64 x 128 256 with 32 768-token histories: 61 -> 39 us).
#include "plh_device.h"
#include "plh_kernels.h"

#include <algorithm>

namespace plh {

namespace {

constexpr int kProcChunk = 4096;
constexpr int kAhead = 4;
constexpr int kQuads = kProcChunk / (4 * kThreads);  // groups of four tokens per thread

// Four consecutive tokens, aligned to their element only: rows of an odd
// vocabulary start anywhere.
template <typename T>
struct Quad;
template <>
struct Quad<float> {
  typedef float V __attribute__((ext_vector_type(4))) __attribute__((aligned(4)));
  V v;
  __device__ __forceinline__ void load(const float* p) { v = *reinterpret_cast<const V*>(p); }
  __device__ __forceinline__ void store(float* p) const { *reinterpret_cast<V*>(p) = v; }
  __device__ __forceinline__ float get(int i) const { return v[i]; }
  __device__ __forceinline__ void set(int i, float x) { v[i] = x; }
};
template <>
struct Quad<double> {
  typedef double V __attribute__((ext_vector_type(2))) __attribute__((aligned(8)));
  V a, b;
  __device__ __forceinline__ void load(const double* p) {
    a = *reinterpret_cast<const V*>(p);
    b = *reinterpret_cast<const V*>(p + 2);
  }
  __device__ __forceinline__ void store(double* p) const {
    *reinterpret_cast<V*>(p) = a;
    *reinterpret_cast<V*>(p + 2) = b;
  }
  __device__ __forceinline__ double get(int i) const { return i < 2 ? a[i & 1] : b[i & 1]; }
  __device__ __forceinline__ void set(int i, double x) {
    if (i < 2) a[i & 1] = x;
    else b[i & 1] = x;
  }
};

// The first n of the four (all of them where n >= 4).
template <typename T>
__device__ __forceinline__ void load(Quad<T>& q, const T* p, int n) {
  if (n >= 4) {
    q.load(p);
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < n) q.set(e, p[e]);
  }
}
template <typename T>
__device__ __forceinline__ void store(const Quad<T>& q, T* p, int n) {
  if (n >= 4) {
    q.store(p);
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < n) p[e] = q.get(e);
  }
}

struct RowRules {
  double r, f, p;
  const double* bias;  // the row's bias list
};

// The value of a token with history word `w` (bit 0: in the history; above it
// the count among the outputs, twice) and bias slot `s` (1 + its place in the
// list, 0: none).  float64, rounded once on return.
template <typename T>
__device__ __forceinline__ T touched(T x, uint32_t w, uint32_t s, const RowRules& q) {
  double v = (double)x;
  if (s != 0) v += q.bias[s - 1];
  if (w != 0) v = v > 0.0 ? v / q.r : v * q.r;
  if (w > 1) v -= q.f * (double)(w >> 1) + q.p;
  return (T)v;
}

// INPLACE: out is x, and only quads that change are read and written.
template <typename T, bool INPLACE>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(sizeof(T) == 4 ? 8 : 6))) void k_process(ProcessArgs a) {
  __shared__ __align__(16) uint32_t words[kProcChunk];  // history words (touched())
  __shared__ __align__(16) uint32_t slots[kProcChunk];  // bias slots
  const int c0 = blockIdx.x * kProcChunk;
  const int ntok = min(kProcChunk, a.V - c0);
  for (int row = blockIdx.y; row < a.B; row += gridDim.y) {
    const T* x = static_cast<const T*>(a.x) + (int64_t)row * a.ld + c0;
    T* o = static_cast<T*>(a.out) + (int64_t)row * a.out_ld + c0;
    RowRules q{a.rep != nullptr ? a.rep[row] : 1.0, a.freq != nullptr ? a.freq[row] : 0.0,
               a.pres != nullptr ? a.pres[row] : 0.0, nullptr};
    int64_t h0 = 0, h1 = 0, out0 = 0, b0 = 0, b1 = 0;
    if (a.hist_off != nullptr) {
      h0 = a.hist_off[a.hist_spans ? 2 * (int64_t)row : row];
      h1 = a.hist_off[a.hist_spans ? 2 * (int64_t)row + 1 : row + 1];
      out0 = a.out_start != nullptr ? h0 + a.out_start[row] : h0;
    }
    if (a.bias_off != nullptr) {
      b0 = a.bias_off[row];
      b1 = a.bias_off[row + 1];
      q.bias = a.bias + b0;
    }
    const bool pen = h1 > h0 && (q.r != 1.0 || q.f != 0.0 || q.p != 0.0);
    const bool bias = b1 > b0;
    const uint32_t* mask = nullptr;
    if (a.mask != nullptr) {
      const int m = a.mask_row != nullptr ? a.mask_row[row] : row;
      if (m >= 0 && m < a.mask_rows) mask = a.mask + (int64_t)m * a.mask_ld;
    }
    if (INPLACE && !pen && !bias && mask == nullptr) continue;

    // the first tokens of the history and of the bias list ahead of the logits: loads
    // return in order, and the tables are built while the logits are on their way
    // (past the end: the last token again, not counted)
    uint32_t id[kAhead], bid = 0;
    if (pen) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) id[u] = (uint32_t)a.hist_ids[min(h0 + threadIdx.x + u * kThreads, h1 - 1)];
    }
    if (bias) bid = (uint32_t)a.bias_ids[min(b0 + threadIdx.x, b1 - 1)];
    __builtin_amdgcn_sched_barrier(0);
    Quad<T> v[kQuads];
    uint32_t allow[kQuads];
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      const int t = 4 * (i * kThreads + (int)threadIdx.x);
      allow[i] = 15u;
      if (t < ntok) {
        if (mask != nullptr) allow[i] = (mask[(uint32_t)(c0 + t) >> 5] >> (t & 31)) & 15u;
        if (!INPLACE) load(v[i], x + t, ntok - t);
      }
    }
    if (pen || bias) {
      for (int i = threadIdx.x; i < (ntok + 3) / 4; i += kThreads) {
        if (pen) reinterpret_cast<uint4*>(words)[i] = uint4{0, 0, 0, 0};
        if (bias) reinterpret_cast<uint4*>(slots)[i] = uint4{0, 0, 0, 0};
      }
      wg_barrier();
      if (pen) {
        for (int64_t h = h0 + threadIdx.x;;) {
#pragma unroll
          for (int u = 0; u < kAhead; ++u) {
            const uint32_t t = id[u] - (uint32_t)c0;
            if (t < (uint32_t)ntok && h + u * kThreads < h1) {
              if (h + u * kThreads >= out0) lds_add(&words[t], 2u);
              else lds_or(&words[t], 1u);
            }
          }
          h += kAhead * kThreads;
          if (h >= h1) break;
#pragma unroll
          for (int u = 0; u < kAhead; ++u) id[u] = (uint32_t)a.hist_ids[min(h + u * kThreads, h1 - 1)];
        }
      }
      if (bias) {
        for (int64_t j = b0 + threadIdx.x; j < b1; j += kThreads) {
          const uint32_t t = (j < b0 + kThreads ? bid : (uint32_t)a.bias_ids[j]) - (uint32_t)c0;
          if (t < (uint32_t)ntok) lds_max(reinterpret_cast<int*>(&slots[t]), (int)(j - b0) + 1);  // the last counts
        }
      }
      wg_barrier();
    }
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      const int t = 4 * (i * kThreads + (int)threadIdx.x);
      if (t >= ntok) break;
      uint4 w{0, 0, 0, 0}, s{0, 0, 0, 0};
      if (pen) w = reinterpret_cast<const uint4*>(words)[t / 4];
      if (bias) s = reinterpret_cast<const uint4*>(slots)[t / 4];
      const uint32_t any = w.x | w.y | w.z | w.w | s.x | s.y | s.z | s.w;
      if (INPLACE) {
        if (any == 0 && allow[i] == 15u) continue;
        if (allow[i] != 0) load(v[i], x + t, ntok - t);
      }
      if (any != 0) {
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if ((ww[e] | ss[e]) != 0 && ((allow[i] >> e) & 1u)) v[i].set(e, touched(v[i].get(e), ww[e], ss[e], q));
      }
      if (allow[i] != 15u) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (((allow[i] >> e) & 1u) == 0) v[i].set(e, (T)-INFINITY);
      }
      store(v[i], o + t, ntok - t);
    }
    wg_barrier();  // the tables are read before the next row clears them
  }
}

// A thread per row: one load behind another, B of them.
template <typename T>
__global__ __launch_bounds__(256) void k_token_logits(const T* x, int64_t ld, int B, int V, const int32_t* ids, T* out) {
  const int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (b >= B) return;
  const int id = ids[b];
  out[b] = (unsigned)id < (unsigned)V ? x[b * ld + id] : (T)NAN;
}

}  // namespace

hipError_t launch_token_logits(const void* x, bool f64, int64_t ld, int B, int V, const int32_t* ids, void* out,
                               hipStream_t s) {
  const dim3 grid((unsigned)(((int64_t)B + 255) / 256));
  if (f64)
    hipLaunchKernelGGL(k_token_logits<double>, grid, dim3(256), 0, s, static_cast<const double*>(x), ld, B, V, ids,
                       static_cast<double*>(out));
  else
    hipLaunchKernelGGL(k_token_logits<float>, grid, dim3(256), 0, s, static_cast<const float*>(x), ld, B, V, ids,
                       static_cast<float*>(out));
  return hipGetLastError();
}

hipError_t launch_process(const ProcessArgs& a, bool f64, hipStream_t s) {
  const dim3 grid((unsigned)(((int64_t)a.V + kProcChunk - 1) / kProcChunk), std::min(a.B, 65535));
  const bool inplace = a.x == a.out;
  if (f64) {
    if (inplace) hipLaunchKernelGGL((k_process<double, true>), grid, dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL((k_process<double, false>), grid, dim3(kThreads), 0, s, a);
  } else {
    if (inplace) hipLaunchKernelGGL((k_process<float, true>), grid, dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL((k_process<float, false>), grid, dim3(kThreads), 0, s, a);
  }
  return hipGetLastError();
}

}  // namespace plh
