// gfx950 kernels for products with e4m3 weights and a scale for each block of
// 128 (plh_fp8_*): out[n, v] = sum_b t[v / 128, b] sum_{k in b} a[n, k] w[v, k], a
// the rows' rounded values.
//
//   k_fp8_act       rows -> RMSNorm -> rounded to e4m3 by blocks -> bf16
//   k_fp8_skinny    at most 32 rows: bound by one read of the codes
//   k_fp8_tiles     more rows (k_fp8_sum: where k is cut into slices)
//   k_fp8_pack, k_fp8_quantize   the weights' layout, once
//
// The products run on the bf16 matrix cores.  The 8-bit ones align a sum's
// products to the largest with 14 bits below it: a block's sum comes out 1.5e-5
// (relative, normal operands) from its exact value, and 4.6e-5 with operands of
// mixed sizes, where bf16 operands give 9e-9 and 8e-8, as float32 sums do.  An
// e4m3 value is a bf16 value, and so is one times its row's scale, a power of two:
// the activations are stored as bf16 with their scales applied, the weights stay
// 8-bit in memory and are widened in registers (one instruction for two), and only
// the weights' scale, the same for a block's 128 x 128, is left for the
// accumulators: one float32 multiply-add for each output and block.
//
// The weights are the matrix instruction's rows and the activations its columns: a
// lane then holds four consecutive v of one n, and the logits leave in 16-byte
// stores.
//
// Layout of the codes: tiles of 32 rows x 128 k, all blocks of 32 rows one after
// the other, each tile 4 KB in the order in which a wave reads it for the 32 x 32
// x 16 instruction: 16-byte piece (q, h, r) of row r and k = 32 q + 16 h + 0 .. 15
// at 1024 q + 512 h + 16 r.  A wave's load is 1 KB of consecutive bytes and 32
// rows are one stream.  (An instruction sums over its k, so any order of k that
// both operands share is right: its two steps of a piece take 8 codes each.)
#include "plh_device.h"
#include "plh_kernels.h"

#include "pagellm_hip.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>

namespace plh {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4e __attribute__((ext_vector_type(4))) __attribute__((aligned(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kBlock = 128;
constexpr int kTileRows = 32;                     // rows of a tile of codes
constexpr int kTileBytes = kTileRows * kBlock;    // its size
constexpr float kE4m3Max = 448.0f;

// n up to 2^31 - 1: the sums would pass an int
__host__ __device__ constexpr int blocks_of(int n) { return (int)(((unsigned)n + kBlock - 1) / kBlock); }
__host__ __device__ constexpr int tiles_of(int n, int rows = kTileRows) {
  return (int)(((unsigned)n + (unsigned)rows - 1) / (unsigned)rows);
}

// Where the 16 codes of row r and k = 16 p .. 16 p + 15 lie, in a matrix of kb
// blocks a row.
__device__ __forceinline__ size_t code_at(int64_t r, int p, int kb) {
  return ((size_t)(r / kTileRows) * kb + p / 8) * kTileBytes + (p % 8) * (kTileRows * 16) + (r % kTileRows) * 16;
}

// Where the 8 rounded values of row n and k = 8 p .. 8 p + 7 lie (16-byte units)
// among the rows' tiles of R rows x 128 k, R that of the matrix instruction: its
// step's operand is 64 lanes x 16 bytes.  p's bits of a block are (q, h, j) as
// above: with R = 32 step (q, j) holds (h, row) in lane 32 h + row, with R = 16 a
// step holds two of the q: step (q / 2, j), lane 16 (2 (q % 2) + h) + row.
template <int R>
__device__ __forceinline__ size_t act_at(int64_t n, int p, int kb) {
  const int q = (p >> 2) & 3, h = (p >> 1) & 1, j = p & 1, r = (int)(n % R);
  const int in = R == 32 ? (2 * q + j) * 64 + 32 * h + r : ((q & 2) + j) * 64 + 16 * (2 * (q & 1) + h) + r;
  return ((size_t)(n / R) * kb + p / 16) * (R * 16) + in;
}

// The smallest power of two s >= 2^-126 with amax <= 448 s (448 = 1.75 * 2^8);
// 1 where amax is not finite.  1 / s is a power of two too, so y / s is exact.
__device__ __forceinline__ float block_scale(float amax) {
  const uint32_t u = __float_as_uint(amax);
  if (u >= 0x7f800000u) return 1.0f;
  const int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float((uint32_t)max(e, 1) << 23);
}

__device__ __forceinline__ float inverse_pow2(float s) { return __uint_as_float(0x7f000000u - __float_as_uint(s)); }

// Four values, |x| <= 448 or NaN for what is not finite, as e4m3 codes.
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

__device__ __forceinline__ float code_input(float y, float inv) {
  const float t = y * inv;
  return fabsf(t) <= kE4m3Max ? t : NAN;
}

template <typename T>
__device__ __forceinline__ float widen(T v) { return (float)v; }

// ------------------------------------------------------------ activations

constexpr int kRun = 8;                    // k values of a thread at a time: one 16-byte piece of the operand
constexpr int kSweep = kRun * kThreads;    // k values of a workgroup at a time
constexpr int kKept = 2;                   // sweeps that stay in registers between the two passes

// Eight values from k0 on, zeros from D on.  Rows start anywhere.
template <typename TX>
__device__ __forceinline__ void load_run(const TX* x, int k0, int D, float (&v)[kRun]) {
  struct __attribute__((packed, aligned(sizeof(TX)))) Run {
    TX e[kRun];
  };
  if (k0 + kRun <= D) {
    const Run r = *reinterpret_cast<const Run*>(x + k0);
#pragma unroll
    for (int j = 0; j < kRun; ++j) v[j] = widen(r.e[j]);
  } else {
#pragma unroll
    for (int j = 0; j < kRun; ++j) v[j] = k0 + j < D ? widen(x[k0 + j]) : 0.0f;
  }
}

// e4m3 codes back to the values they stand for, times the power of two s, as
// bf16 (exact: four significant bits).
__device__ __forceinline__ uint32_t rounded2(uint32_t codes, bool hi, float s) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 v = hi ? __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false);
  return (__float_as_uint(v[0] * s) >> 16) | (__float_as_uint(v[1] * s) & 0xffff0000u);
}

// The largest of a row of 16 lanes, in all of them (rotations within the row).
__device__ __forceinline__ float row16_max(float v) {
  v = fmaxf(v, dpp<0x128, 0xf>(v, v));
  v = fmaxf(v, dpp<0x124, 0xf>(v, v));
  v = fmaxf(v, dpp<0x122, 0xf>(v, v));
  return fmaxf(v, dpp<0x121, 0xf>(v, v));
}

// One workgroup per row, more than 2^20 rows in turn (a grid holds 2^32 threads); a
// block's 16 threads are one row of 16 lanes.  The norm is computed in float64: a last
// bit of y next to a border between two codes would change the code.  8 x 4096 float32
// 5 us (its chain of loads and sums), 2048 x 4096 bf16 23-24 us (the 16-byte stores of the
// operand's layout, 512 bytes apart).
template <typename TX, int R>
__global__ __launch_bounds__(kThreads) void k_fp8_act(Fp8Args a) {
  __shared__ double red[kWaves];
  const int kt = threadIdx.x * kRun;
  for (int64_t n = blockIdx.x; n < a.N; n += gridDim.x) {
    const TX* x = static_cast<const TX*>(a.x) + n * a.ldx;
    float v[kKept][kRun], w[kKept][kRun];
#pragma unroll
    for (int i = 0; i < kKept; ++i) {
      load_run(x, kt + i * kSweep, a.D, v[i]);
      if (a.norm != nullptr) load_run(a.norm, kt + i * kSweep, a.D, w[i]);
    }
    double r = 1.0;
    if (a.norm != nullptr) {
      double s = 0.0;
#pragma unroll
      for (int i = 0; i < kKept; ++i)
#pragma unroll
        for (int j = 0; j < kRun; ++j) s += (double)v[i][j] * (double)v[i][j];
      for (int k0 = kt + kKept * kSweep; k0 < a.D; k0 += kSweep) {
        float u[kRun];
        load_run(x, k0, a.D, u);
#pragma unroll
        for (int j = 0; j < kRun; ++j) s += (double)u[j] * (double)u[j];
      }
      s = block_sum(s, red);
      r = 1.0 / sqrt(s / (double)a.D + a.eps);
    }
    const auto emit = [&](int k0, float (&y)[kRun], const float (&g)[kRun]) {
      float amax = 0.0f;
#pragma unroll
      for (int j = 0; j < kRun; ++j) {
        if (a.norm != nullptr) y[j] = k0 + j < a.D ? (float)((double)y[j] * r * (double)g[j]) : 0.0f;
        amax = fmaxf(amax, fabsf(y[j]));
      }
      const float s = block_scale(row16_max(amax)), inv = inverse_pow2(s);
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t c = codes4(code_input(y[4 * j], inv), code_input(y[4 * j + 1], inv), code_input(y[4 * j + 2], inv),
                                  code_input(y[4 * j + 3], inv));
        o[2 * j] = rounded2(c, false, s);
        o[2 * j + 1] = rounded2(c, true, s);
      }
      a.act[act_at<R>(n, k0 / kRun, a.kb)] = uint4{o[0], o[1], o[2], o[3]};
    };
#pragma unroll
    for (int i = 0; i < kKept; ++i)
      if (kt + i * kSweep < a.kb * kBlock) emit(kt + i * kSweep, v[i], w[i]);
    for (int k0 = kt + kKept * kSweep; k0 < a.kb * kBlock; k0 += kSweep) {
      load_run(x, k0, a.D, v[0]);
      if (a.norm != nullptr) load_run(a.norm, k0, a.D, w[0]);
      emit(k0, v[0], w[0]);
    }
  }
}

// ----------------------------------------------------------------- product

// Eight codes as the matrix instruction's operand.
__device__ __forceinline__ bf16x8 widen8(uint32_t lo, uint32_t hi) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ bf16x8 as_bf16(u32x4 v) { return __builtin_bit_cast(bf16x8, v); }

// The matrix instruction with R rows of weights and R of activations, and its
// operands of one tile and block.
template <int R>
struct Mma;
template <>
struct Mma<32> {
  typedef f32x16 Acc;
  static constexpr int kSteps = 8;    // per block of 128
  static constexpr int kPieces = 4;   // 16-byte pieces of codes a lane holds
  static __device__ __forceinline__ size_t piece(int i) { return (size_t)i * 1024 + lane() * 16; }
  static __device__ __forceinline__ Acc mma(bf16x8 w, bf16x8 x, Acc c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(w, x, c, 0, 0, 0);
  }
  // accumulator registers 4 g .. 4 g + 3 hold rows row(g) .. + 3 of column lane() % 32
  static __device__ __forceinline__ int row(int g) { return 8 * g + 4 * (lane() >> 5); }
};
template <>
struct Mma<16> {
  typedef f32x4 Acc;
  static constexpr int kSteps = 4;
  static constexpr int kPieces = 2;
  // of 16 rows of a tile, the others 256 bytes further on: lane group g reads
  // (q, h) = (2 i + g / 2, g % 2)
  static __device__ __forceinline__ size_t piece(int i) {
    const int g = lane() >> 4;
    return (size_t)(2 * i + (g >> 1)) * 1024 + (g & 1) * 512 + (lane() & 15) * 16;
  }
  static __device__ __forceinline__ Acc mma(bf16x8 w, bf16x8 x, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x, c, 0, 0, 0);
  }
  static __device__ __forceinline__ int row(int g) { return 4 * (lane() >> 4); }
};

// Four consecutive logits of row n, those inside the vocabulary.
__device__ __forceinline__ void store4(const Fp8Args& a, int n, int v, f32x4 t) {
  if (n >= a.N || v >= a.V) return;
  float* o = a.out + (int64_t)n * a.ldo + v;
  if (v + 4 <= a.V) {
    *reinterpret_cast<f32x4e*>(o) = t;
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (v + e < a.V) o[e] = t[e];
  }
}

// --------------------------------------------------------------- few rows

// Bound by the read of the codes: 8 x 4096 x 128 256 92 us, 5.8 TB/s (a large copy
// moves 4.95 TB/s here).
constexpr int kSkinnyCols = 64;  // columns of the logits of a workgroup: half a scale block

// R rows x 64 columns per workgroup.  The 8 waves share them and take every
// eighth block of k each, codes and activations straight from memory into
// registers; their sums meet in LDS at the end, in a fixed order.
template <int R>
__global__ __launch_bounds__(kThreads) void k_fp8_skinny(Fp8Args a) {
  using M = Mma<R>;
  constexpr int kVT = kSkinnyCols / R, kRegs = R * R / 64, kQuads = kVT * kRegs / 4;
  __shared__ f32x4 sm[kWaves][kQuads][kWave];
  const int v0 = blockIdx.x * kSkinnyCols;
  typename M::Acc acc[kVT];
#pragma unroll
  for (int i = 0; i < kVT; ++i) acc[i] = typename M::Acc{};
  const uint8_t* w[kVT];
  // rows past the last read as the last ones, and are not stored
#pragma unroll
  for (int i = 0; i < kVT; ++i) {
    const int v = min(v0 + i * R, tiles_of(a.V) * kTileRows - R);
    w[i] = a.codes + (size_t)(v / kTileRows) * a.kb * kTileBytes + (v % kTileRows) * 16;
  }
  const u32x4* act = reinterpret_cast<const u32x4*>(a.act) + lane();
  const float* ts = a.scales + (size_t)(v0 / kBlock) * a.kb;
  for (int b = wave(); b < a.kb; b += kWaves) {
    u32x4 x[M::kSteps], c[kVT][M::kPieces];
#pragma unroll
    for (int i = 0; i < kVT; ++i)
#pragma unroll
      for (int q = 0; q < M::kPieces; ++q)
        c[i][q] = *reinterpret_cast<const u32x4*>(w[i] + (size_t)b * kTileBytes + M::piece(q));
#pragma unroll
    for (int s = 0; s < M::kSteps; ++s) x[s] = act[(size_t)b * (R * 16) + s * kWave];
    const float t = ts[b];
#pragma unroll
    for (int i = 0; i < kVT; ++i) {
      typename M::Acc p{};
#pragma unroll
      for (int q = 0; q < M::kPieces; ++q) {
        p = M::mma(widen8(c[i][q][0], c[i][q][1]), as_bf16(x[2 * q]), p);
        p = M::mma(widen8(c[i][q][2], c[i][q][3]), as_bf16(x[2 * q + 1]), p);
      }
#pragma unroll
      for (int e = 0; e < kRegs; ++e) acc[i][e] = fmaf(p[e], t, acc[i][e]);
    }
  }
#pragma unroll
  for (int i = 0; i < kVT; ++i)
#pragma unroll
    for (int g = 0; g < kRegs / 4; ++g)
      sm[wave()][i * (kRegs / 4) + g][lane()] =
          f32x4{acc[i][4 * g], acc[i][4 * g + 1], acc[i][4 * g + 2], acc[i][4 * g + 3]};
  wg_barrier();
  for (int u = wave(); u < kQuads; u += kWaves) {
    f32x4 t = sm[0][u][lane()];
#pragma unroll
    for (int k = 1; k < kWaves; ++k) t += sm[k][u][lane()];
    store4(a, lane() % R, v0 + u / (kRegs / 4) * R + M::row(u % (kRegs / 4)), t);
  }
}

// -------------------------------------------------------------- more rows

// The tile of a workgroup.  kGroup row tiles run under one column tile, then the
// next.  With `ranges`, the workgroups of one XCD (every eighth) get one contiguous
// range of that order, so that they share codes and activations in its L2 (50 257
// columns: 256 rows of 4096 119 -> 113 us, 1024 rows 433 -> 419 us); without, the
// whole chip writes neighbouring tiles of the logits, which counts for more where a
// tile's sums are short and the rows many (2048 rows of 512: 217 -> 199 us, of 1000
// 297 -> 278 us, of 1536 375 -> 365 us, of 2048 458 us either way).
constexpr int kXcds = 8, kGroup = 8;
constexpr int kPlainRows = 1024, kPlainBlocks = 16;
__device__ __forceinline__ void tile_of_group(int vtiles, int ntiles, bool ranges, int& vt, int& nt) {
  const int total = vtiles * ntiles, x = blockIdx.x % kXcds, slot = blockIdx.x / kXcds;
  const int idx = ranges ? x * (total / kXcds) + min(x, total % kXcds) + slot : (int)blockIdx.x;
  const int g = idx / (kGroup * vtiles), in = idx % (kGroup * vtiles), rows = min(kGroup, ntiles - g * kGroup);
  vt = in / rows;
  nt = g * kGroup + in % rows;
}

// instruction classes of __builtin_amdgcn_sched_group_barrier
constexpr int kVector = 0x002, kMatrix = 0x008, kDsRead = 0x100;

// A workgroup's 8 waves lie WN along the rows; each forms VI x 2 tiles of 32
// columns x 32 rows.  Codes go from memory into registers, one block ahead,
// activations through LDS, double-buffered, staged in registers one block ahead:
// a wave reads 64 rows' activations from LDS for VI * 32 columns, and only the WN
// waves side by side widen the same codes.  Block sums are their own registers, so
// that a block's scale meets its sum: as many again as the accumulators, which
// keeps a wave's tile at 64 x 64.
//
// Bound by the matrix cores at the clock that the power limit leaves them (1.9 GHz; operands
// of zeros run a fifth faster), 53% busy: 256 x 4096 x 128 256 263-274 us, 2048 x 4096 x
// 32 000 493-520 us (1.03-1.09 PFLOP/s; a large bf16 matrix product reaches 1.2 here); 33,
// 64 and 128 rows x 4096 x 128 256 109, 117 and 152 us.  What it
// took there: loads issued where they are wanted (582 -> 540 us: the compiler sinks
// them to their use), LDS reads and vector instructions placed among the products
// (-> 532), three LDS buffers instead of two (256 rows: 283 -> 274), whole runs of
// output (2048 x 1000 x 50 257: 358 -> 308).  Two workgroups of four waves a CU are no
// faster (128 x 128 outputs each: 576, 256 x 64: 533).
template <int VI, int WN, int NW>
struct Tiles {
  static constexpr int kCols = NW / WN * VI * 32;  // of a workgroup
  static constexpr int kRows = WN * 64;
  static constexpr int kStage = kRows / 32;        // 32-row tiles of activations in LDS
  static constexpr int kUnit = kTileRows * 16;     // 16-byte units of such a tile and block
  static constexpr int kLoads = kStage * kUnit / (NW * kWave);  // of a thread
  static_assert(kLoads <= Mma<32>::kSteps / 2, "a step of every two stores one");
};

template <int VI, int WN, int NW>
__global__ __launch_bounds__(NW * kWave) __attribute__((amdgpu_waves_per_eu(VI == 2 ? 2 : 4, VI == 2 ? 2 : 4))) void
k_fp8_tiles(Fp8Args a) {
  using G = Tiles<VI, WN, NW>;
  using M = Mma<32>;
  constexpr int kUnit = G::kUnit, kN = NW * kWave;
  __shared__ u32x4 sm[3][G::kStage * kUnit];
  int vt, nt;
  tile_of_group(tiles_of(a.V, G::kCols), tiles_of(a.N, G::kRows), a.N <= kPlainRows || a.kb >= kPlainBlocks, vt, nt);
  const int w = uniform(wave()), l = lane();
  const int v0 = vt * G::kCols + w / WN * (VI * 32), n0 = nt * G::kRows, nw = w % WN * 64;
  const int b0 = (int)((int64_t)a.kb * blockIdx.z / gridDim.z), b1 = (int)((int64_t)a.kb * (blockIdx.z + 1) / gridDim.z);
  // tiles past the last read as the last, and are not stored
  const uint8_t* codes[VI];
#pragma unroll
  for (int i = 0; i < VI; ++i)
    codes[i] = a.codes + (size_t)min(v0 / kTileRows + i, tiles_of(a.V) - 1) * a.kb * kTileBytes;
  const u32x4* act[G::kLoads];
#pragma unroll
  for (int r = 0; r < G::kLoads; ++r) {
    const int at = r * kN + (int)threadIdx.x;
    act[r] = reinterpret_cast<const u32x4*>(a.act) +
             (size_t)min(n0 / kTileRows + at / kUnit, tiles_of(a.N) - 1) * a.kb * kUnit + at % kUnit;
  }
  const float* ts = a.scales + (size_t)min(v0 / kBlock, blocks_of(a.V) - 1) * a.kb;

  u32x4 c[VI][M::kPieces], st[G::kLoads];
  f32x16 acc[VI][2], p[VI][2];
#pragma unroll
  for (int i = 0; i < VI; ++i) {
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = f32x16{}, p[i][j] = f32x16{};
#pragma unroll
    for (int q = 0; q < M::kPieces; ++q)
      c[i][q] = *reinterpret_cast<const u32x4*>(codes[i] + (size_t)b0 * kTileBytes + M::piece(q));
  }
  // activations of block b in buffer (b - b0) % 3: two blocks ahead when the loop
  // is at one, and a third in registers
  auto load = [&](int b, int r) { return act[r][(size_t)min(b, b1 - 1) * kUnit]; };
#pragma unroll
  for (int r = 0; r < G::kLoads; ++r) sm[0][r * kN + (int)threadIdx.x] = load(b0, r);
#pragma unroll
  for (int r = 0; r < G::kLoads; ++r) sm[1][r * kN + (int)threadIdx.x] = load(b0 + 1, r);
#pragma unroll
  for (int r = 0; r < G::kLoads; ++r) st[r] = load(b0 + 2, r);
  wg_barrier();
  const int x0 = nw / 32 * kUnit + l;
  float t = 0.0f;  // the scale of the block before
  bf16x8 x[2][2], wt[2][VI];
#pragma unroll
  for (int j = 0; j < 2; ++j) x[0][j] = as_bf16(sm[0][x0 + j * kUnit]);
#pragma unroll
  for (int i = 0; i < VI; ++i) wt[0][i] = widen8(c[i][0][0], c[i][0][1]);
  int at = 0;  // this block's buffer
  for (int b = b0; b < b1; ++b) {
    const int next = min(b + 1, b1 - 1), after = at == 2 ? 0 : at + 1, last = at == 0 ? 2 : at - 1;
    const float tb = ts[b];
#pragma unroll
    for (int s = 0; s < M::kSteps; ++s) {
      // the next step's operands, and the next block's codes into registers that
      // have been widened
      const int n = (s + 1) % M::kSteps;
      const u32x4* xs = &sm[n == 0 ? after : at][x0 + n * kWave];
#pragma unroll
      for (int j = 0; j < 2; ++j) x[n & 1][j] = as_bf16(xs[j * kUnit]);
#pragma unroll
      for (int i = 0; i < VI; ++i) wt[n & 1][i] = widen8(c[i][n / 2][n % 2 * 2], c[i][n / 2][n % 2 * 2 + 1]);
      if (s % 2 == 0) {
#pragma unroll
        for (int i = 0; i < VI; ++i)
          c[i][s / 2] = *reinterpret_cast<const u32x4*>(codes[i] + (size_t)next * kTileBytes + M::piece(s / 2));
      }
      // the block two ahead into the buffer that was read last
      if (s % 2 == 1 && s / 2 < G::kLoads) {
        sm[last][s / 2 * kN + (int)threadIdx.x] = st[s / 2];
        st[s / 2] = load(b + 3, s / 2);
      }
#pragma unroll
      for (int i = 0; i < VI; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (s == 0) {
            // the block before meets its scale among this one's first products
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = fmaf(p[i][j][e], t, acc[i][j][e]);
            p[i][j] = f32x16{};
          }
          p[i][j] = M::mma(wt[s & 1][i], x[s & 1][j], p[i][j]);
        }
      // LDS reads first, then the vector instructions among the products
      __builtin_amdgcn_sched_group_barrier(kDsRead, 2, 0);
#pragma unroll
      for (int m = 0; m < 2 * VI; ++m) {
        if (s == 0) __builtin_amdgcn_sched_group_barrier(kVector, 16, 0);
        __builtin_amdgcn_sched_group_barrier(kMatrix, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kVector, 2, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    t = tb;
    at = after;
    wg_barrier();
  }
#pragma unroll
  for (int i = 0; i < VI; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = fmaf(p[i][j][e], t, acc[i][j][e]);
  if (gridDim.z > 1) {
    a.out = a.part + (size_t)blockIdx.z * a.N * a.V;
    a.ldo = a.V;
  }
  // 32 rows at a time through the wave's part of LDS (the last barrier has
  // passed: nobody reads activations there), so that a store writes whole runs of
  // the logits' rows
  constexpr int kRun4 = VI * 8, kPitch = kRun4 + 1;  // 16-byte units of a row, and its pitch
  u32x4* own = &sm[0][0] + w * 32 * kPitch;
  static_assert(NW * 32 * kPitch <= 3 * G::kStage * kUnit, "the waves' parts lie in LDS");
#pragma unroll
  for (int j = 0; j < 2; ++j) {
#pragma unroll
    for (int i = 0; i < VI; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        own[l % 32 * kPitch + 8 * i + M::row(g) / 4] = __builtin_bit_cast(
            u32x4, f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]});
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = 0; r < 32 * kRun4 / kWave; ++r) {
      const int at = r * kWave + l;
      store4(a, n0 + nw + 32 * j + at / kRun4, v0 + at % kRun4 * 4,
             __builtin_bit_cast(f32x4, own[at / kRun4 * kPitch + at % kRun4]));
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// The slices' partial sums, in order.
__global__ __launch_bounds__(256) void k_fp8_sum(Fp8Args a, int slices) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, n = (int64_t)a.N * a.V;
  if (i >= n) return;
  float t = a.part[i];
  for (int z = 1; z < slices; ++z) t += a.part[z * n + i];
  a.out[i / a.V * a.ldo + i % a.V] = t;
}

// ---------------------------------------------------------------- weights

// One thread per 16 codes of the layout, read byte by byte: rows start anywhere.  Once a
// model: 128 256 x 4096 0.8 ms.
__global__ __launch_bounds__(256) void k_fp8_pack(const uint8_t* codes, int64_t ldc, const float* scales, int64_t lds,
                                                  int V, int D, uint8_t* out, float* out_scales) {
  const int kb = blocks_of(D);
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, pieces = (int64_t)tiles_of(V) * kTileRows * kb * 8;
  if (i < pieces) {
    const int64_t r = i / (kb * 8);
    const int q = (int)(i % (kb * 8));
    __align__(16) uint8_t c[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) c[j] = r < V && q * 16 + j < D ? codes[r * ldc + q * 16 + j] : 0;
    *reinterpret_cast<uint4*>(out + code_at(r, q, kb)) = *reinterpret_cast<const uint4*>(c);
  }
  if (i < (int64_t)blocks_of(V) * kb) out_scales[i] = scales[i / kb * lds + i % kb];
}

// One workgroup of 256 threads per block of 128 x 128.  `along_v`: neighbouring threads
// take neighbouring rows (W is contiguous along v).  Once a model: 128 256 x 4096 2.1 ms from
// float32, either way round.
template <typename TW>
__global__ __launch_bounds__(256) void k_fp8_quantize(const TW* W, int64_t sv, int64_t sd, int V, int D, uint8_t* out,
                                                      float* out_scales) {
  __shared__ float tile[kBlock][kBlock + 1];
  __shared__ float red[4];
  const int kb = blocks_of(D), b = blockIdx.x % kb, vb = blockIdx.x / kb;
  const bool along_v = sv < sd;
  float amax = 0.0f;
  for (int i = threadIdx.x; i < kBlock * kBlock; i += 256) {
    const int r = along_v ? i % kBlock : i / kBlock, k = along_v ? i / kBlock : i % kBlock;
    const int64_t v = (int64_t)vb * kBlock + r;
    const int d = b * kBlock + k;
    const float x = v < V && d < D ? widen(W[v * sv + d * sd]) : 0.0f;
    tile[r][k] = x;
    if (fabsf(x) < INFINITY) amax = fmaxf(amax, fabsf(x));
  }
  amax = wave_max(amax);
  if (lane() == 0) red[wave()] = amax;
  __syncthreads();
  const float s = block_scale(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]))), inv = inverse_pow2(s);
  if (threadIdx.x == 0) out_scales[(size_t)vb * kb + b] = s;
  for (int i = threadIdx.x; i < kBlock * 8; i += 256) {
    const int r = i % kBlock, q = i / kBlock;
    if (vb * kBlock + r >= tiles_of(V) * kTileRows) continue;
    uint32_t c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float* t = &tile[r][q * 16 + 4 * j];
      c[j] = codes4(code_input(t[0], inv), code_input(t[1], inv), code_input(t[2], inv), code_input(t[3], inv));
    }
    *reinterpret_cast<uint4*>(out + code_at((int64_t)vb * kBlock + r, b * 8 + q, kb)) = uint4{c[0], c[1], c[2], c[3]};
  }
}

}  // namespace

size_t fp8_codes_bytes(int V, int D) { return (size_t)tiles_of(V) * blocks_of(D) * kTileBytes; }

namespace {
// Rows of the matrix instruction: 16 where that holds all rows, else 32.
int rows_of(int N) { return N <= 16 ? 16 : 32; }

template <int R>
hipError_t launch_act(const Fp8Args& a, int dtype, hipStream_t s) {
  const dim3 grid(std::min(a.N, 1 << 20));
  if (dtype == PLH_BF16) hipLaunchKernelGGL((k_fp8_act<__hip_bfloat16, R>), grid, dim3(kThreads), 0, s, a);
  else if (dtype == PLH_F16) hipLaunchKernelGGL((k_fp8_act<__half, R>), grid, dim3(kThreads), 0, s, a);
  else hipLaunchKernelGGL((k_fp8_act<float, R>), grid, dim3(kThreads), 0, s, a);
  return hipGetLastError();
}
}  // namespace

namespace {
size_t act_bytes(int N, int D) {
  const int R = rows_of(N);
  return (size_t)tiles_of(N, R) * R * blocks_of(D) * kBlock * 2;
}

// How a product of more than 32 rows runs: 128 rows a workgroup where such tiles
// (nearly) fill the chip, one each CU, else 64, two each CU; and the slices that k is
// cut into where the tiles are fewer than the CUs.  (Rows x 4096 x columns, 128 / 64 rows a
// workgroup, us: 1000 x 4000, 128 tiles, 58 / 48; 100 x 16 000, 63 tiles, 37 / 33; 300 x
// 16 000, 189 tiles, 62 / 63; 2048 x 4000, 256 tiles, 80 / 84; 2048 x 16 000 254 /
// 263.  In slices / in one: 100 x 4096 x 4000 23 / 35 us, 100 x 1000 x 16 000 23 /
// 16: a sum of few blocks is done before a second launch could add slices up.)
using WideTiles = Tiles<2, 2, 8>;
using NarrowTiles = Tiles<1, 1, 8>;
constexpr int kSliceFrom = 12;  // blocks of a sum that is cut into slices, of at least four
struct Plan {
  bool wide;
  int tiles, slices;
};

Plan plan_of(int N, int V, int D, int num_cu) {
  const int64_t w = (int64_t)tiles_of(V, WideTiles::kCols) * tiles_of(N, WideTiles::kRows);
  const bool wide = N > 64 && 4 * w >= 3 * (int64_t)num_cu;
  const int64_t t = wide ? w : (int64_t)tiles_of(V, NarrowTiles::kCols) * tiles_of(N, NarrowTiles::kRows);
  const int blocks = blocks_of(D);
  const int64_t s = blocks < kSliceFrom ? 1 : std::min<int64_t>({num_cu / t, blocks / 4, 16});
  return Plan{wide, (int)t, (int)std::max<int64_t>(1, s)};
}
}  // namespace

size_t fp8_ws_bytes(int N, int V, int D, int num_cu) {
  if (N <= 32) return act_bytes(N, D);
  const Plan p = plan_of(N, V, D, num_cu);
  return act_bytes(N, D) + (p.slices > 1 ? (size_t)p.slices * N * V * sizeof(float) : 0);
}

hipError_t launch_fp8_pack(const uint8_t* codes, int64_t ldc, const float* scales, int64_t lds, int V, int D,
                           uint8_t* out_codes, float* out_scales, hipStream_t s) {
  const int64_t pieces = (int64_t)tiles_of(V) * kTileRows * blocks_of(D) * 8;
  hipLaunchKernelGGL(k_fp8_pack, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, s, codes, ldc, scales, lds, V, D,
                     out_codes, out_scales);
  return hipGetLastError();
}

hipError_t launch_fp8_quantize(const void* w, int dtype, int64_t sv, int64_t sd, int V, int D, uint8_t* out_codes,
                               float* out_scales, hipStream_t s) {
  const dim3 grid((unsigned)(blocks_of(V) * (int64_t)blocks_of(D)));
  if (dtype == PLH_BF16)
    hipLaunchKernelGGL((k_fp8_quantize<__hip_bfloat16>), grid, dim3(256), 0, s, static_cast<const __hip_bfloat16*>(w),
                       sv, sd, V, D, out_codes, out_scales);
  else if (dtype == PLH_F16)
    hipLaunchKernelGGL((k_fp8_quantize<__half>), grid, dim3(256), 0, s, static_cast<const __half*>(w), sv, sd, V, D,
                       out_codes, out_scales);
  else
    hipLaunchKernelGGL((k_fp8_quantize<float>), grid, dim3(256), 0, s, static_cast<const float*>(w), sv, sd, V, D,
                       out_codes, out_scales);
  return hipGetLastError();
}

hipError_t launch_fp8_linear(Fp8Args a, int dtype, void* ws, int num_cu, hipStream_t s) {
  a.kb = blocks_of(a.D);
  a.act = static_cast<uint4*>(ws);
  const int R = rows_of(a.N);
  hipError_t e = R == 16 ? launch_act<16>(a, dtype, s) : launch_act<32>(a, dtype, s);
  if (e != hipSuccess) return e;
  if (a.N <= 32) {
    const dim3 grid((a.V + kSkinnyCols - 1) / kSkinnyCols);
    if (R == 16) hipLaunchKernelGGL((k_fp8_skinny<16>), grid, dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL((k_fp8_skinny<32>), grid, dim3(kThreads), 0, s, a);
    return hipGetLastError();
  }
  const Plan p = plan_of(a.N, a.V, a.D, num_cu);
  a.part = reinterpret_cast<float*>(static_cast<char*>(ws) + act_bytes(a.N, a.D));
  const dim3 grid(p.tiles, 1, p.slices);
  if (p.wide) hipLaunchKernelGGL((k_fp8_tiles<2, 2, 8>), grid, dim3(kThreads), 0, s, a);
  else hipLaunchKernelGGL((k_fp8_tiles<1, 1, 8>), grid, dim3(kThreads), 0, s, a);
  e = hipGetLastError();
  if (e != hipSuccess || p.slices == 1) return e;
  hipLaunchKernelGGL(k_fp8_sum, dim3((unsigned)(((int64_t)a.N * a.V + 255) / 256)), dim3(256), 0, s, a, p.slices);
  return hipGetLastError();
}

}  // namespace plh
