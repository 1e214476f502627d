// Softmax cross entropy of a fully connected output layer over a large vocabulary, and its gradient, for gfx950, without
// keeping the logits:
//
//   z = X W^T + bias,  lse_b = log sum_v exp z_bv,  loss_b = lse_b - z_b,label
//   dL_bv = exp(z_bv - lse_b) - [v = label_b],  dX = g dL W,  dW = (g dL)^T X,  db = sum_b g_b dL_b,   g_b = scale dloss_b
//
// The vocabulary is walked in pieces.  Forward: one product per piece whose epilogue reduces each T / 2 classes of a
// row to a maximum and a sum of exponentials; nothing of size [B, V] is written.  Backward: per piece the logits again,
// dL rounded to f16 planes, the two products that read it.  (For memory's sake: for [8192 x 2048] BF16 against 65536 classes the
// logits take 1.7 ms again, where writing and reading 2 GiB of them would take 0.85.)
// Bound by the 16-bit matrix pipe: 2 B K V operations forward, 6 B K V backward, times three for the two planes of an fp32
// input (half_gemm.hpp); by reading W where there are few rows.  [8192 x 2048] BF16 against 65536 classes, forward and
// backward: 8.2 - 8.5 ms = 1035 - 1075 TFLOP/s, packing included; [777 x 1000] FP32 against 30011: 740 - 765 us.
//
// Operands are packed as f16 planes of powers-of-two multiples, each row of X and of W by its own largest magnitude (a
// padding row full of garbage spoils nobody's scale).  bf16 values have 8 bits and one plane holds them exactly, down
// to 2^-30 of their row's largest; fp32 values take two planes, whose second has all its bits down to 2^-18 of that.  f16 ends at
// 2^-24: what is smaller is held to 2^-39 (bf16) or 2^-40 (fp32) of the row's largest.  dL is in [-1, 1] and held times 2^15,
// rounded to 11 bits (bf16; the result keeps 8) where it is above 2^-29, or 22 (fp32) above 2^-18, and to 2^-40 below.
// Where a product's sum runs over rows that are scaled differently (dX over W's, dW over X's), dL carries what undoes the
// scale, as a share of the largest such factor, which multiplies the result.  For dW X is packed times dloss (one more
// rounding for bf16, none without dloss).  Factors more than 2^19 apart would leave few bits to the small ones (a padding row of
// W that was never set, one row of the batch with a huge dloss): a piece where they are, which the device finds out by itself,
// keeps dL in fp32 where its planes would lie and multiplies it with the operands as they are on the fp32 matrix pipe.
#pragma once

#include <algorithm>
#include <cmath>

#include "half_gemm.hpp"

namespace dlmi {

struct CeArgs {
  size_t B, K, V;
  void const *X, *W;
  float const *bias;
  int const *labels;
  float *loss, *lse;
  // backward
  float const *lse_in, *dloss;
  float scale;
  void *dX, *dW;
  float *db;
  int accumulate;
};

template <class T>
int ce_forward(dlmi_ctx *ctx, CeArgs const &a);
template <class T>
int ce_backward(dlmi_ctx *ctx, CeArgs const &a);

#ifdef DLMI_CE_IMPLEMENTATION

constexpr int kCeBlock = 256;
constexpr float kCeDl = 32768.0f;         // dL is held times this

template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) CeOct {
  T v[8];
};

// 2^e with the largest magnitude m times it in [2^14, 2^15); 1 for m = 0, at most 2^126.
__device__ __forceinline__ float ce_scale(float m) {
  if (!(m > 0.0f)) return 1.0f;
  int e = 14 - (static_cast<int>(__float_as_uint(m) >> 23) - 127);
  e = e > 126 ? 126 : e;
  return __uint_as_float(static_cast<unsigned>(e + 127) << 23);
}
// Its inverse: a power of two of at least 2^-126.
__device__ __forceinline__ float ce_unscale(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

__device__ __forceinline__ float ce_finite_max(float m, float x) {
  x = fabsf(x);
  return x <= 3.402823466e+38f && x > m ? x : m;  // infinities and NaN set no scale
}

__device__ __forceinline__ float ce_wave_max(float m) {
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  return m;
}

// What a row counts in the gradient, but for the common factor `scale`.
__device__ __forceinline__ float ce_row_weight(CeArgs const &a, size_t b) {
  int const l = a.labels[b];
  if (l < 0 || static_cast<size_t>(l) >= a.V) return 0.0f;
  return a.dloss != nullptr ? a.dloss[b] : 1.0f;
}

// The largest of n values, the same in all lanes of a wavefront.
__device__ __forceinline__ float ce_largest(float const *v, unsigned n, int lane) {
  float m = 0.0f;
#pragma unroll 16
  for (unsigned q = lane; q < n; q += 64) m = fmaxf(m, v[q]);
  return ce_wave_max(m);
}

// Whether factors that undo scales lie far apart: the largest of them times the largest scale (the smallest factor's inverse).
// Up to here a row's terms keep an absolute error of 2^-40 of the largest factor's, 2^-21 of their own factor's.  (Of 8192 normal
// dloss one batch in twenty has a value this close to 0; at 2^16 it would be one in three.)
__device__ __forceinline__ bool ce_apart(float const *most, float const *finest) { return most[0] * finest[0] > 524288.0f; }

// Rows of src [rows, cols], each scaled by its own largest magnitude and packed as it stands (`as`: row r, k = c) and / or
// transposed (`across`: row c, k = r), padding zero.  unscale[r]: the inverse scale of `as`, unscale_across[r] that of
// `across` (padding rows have entries too).  LABELS (X): `across` holds the row times ce_row_weight, scaled by its own
// largest, and zeros in rows left out; otherwise (W) the two are the same.  The largest unscale_across of a piece of W and its
// largest scale go to most.w[piece] and most.w[pieces + piece] by an integer maximum in memory (positive floats order like
// integers, and no order changes a maximum), which packing X has cleared; X's are left per workgroup and joined by the first
// workgroup that packs W.
// The four wavefronts of a workgroup share the columns of 8 rows at a time, a lane 8 columns of one of them; up to KEEP
// octets of a lane stay in registers between the search for the largest and the packing (wider rows are read twice).  An
// octet is a piece of a fragment as it stands; for the transposed ones the wavefront turns 8 x 64 values through 2 KiB of
// LDS that only it uses.  [30011 x 1000] FP32: 46 us one way, 67 both = 5.3 - 5.5 TB/s.
// ALONE: rows of up to 64 KEEP columns, a wavefront takes 8 of its own, all their columns ([96475 x 119] BF16: 66 -> 18 us).
constexpr unsigned kCePackBlocks = 1024;

// (All null in the forward pass.)
struct CeMost {
  float *w;          // of each piece: the largest factors, then the largest scales
  float *x, *parts;  // the same two of X; of its packing workgroups
  unsigned nparts, piece, pieces;
};

template <class T, int NP, int KEEP, bool LABELS, bool ALONE>
__global__ __launch_bounds__(kCeBlock) void k_ce_pack(CeArgs a, T const *src, size_t rows, size_t padded, size_t cols, unsigned kblocks_as,
                                                      unsigned kblocks_across, float *unscale, float *unscale_across, CeMost most, char *as, char *across) {
  __shared__ float turn[4][8][68];
  __shared__ float top[2][4][8];
  int const lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int const r8 = lane >> 3, c8 = (lane & 7) * 8;
  unsigned const tiles = kblocks_as / 4;  // of 64 columns, padding included
  unsigned const step = ALONE ? 1 : 4, first = ALONE ? 0 : wave;  // of a wavefront's tiles
  bool const narrow = cols < 8, kept = ALONE || (tiles + 3) / 4 <= KEEP;
  float mine = 0.0f, finest = 0.0f;
  int flip = 0;
  size_t const at = ALONE ? static_cast<size_t>(blockIdx.x) * 4 + wave : blockIdx.x, stride = static_cast<size_t>(gridDim.x) * (ALONE ? 4 : 1);
  for (size_t r0 = at * 8; r0 < padded; r0 += stride * 8) {
    size_t const r = r0 + r8;
    T const *const row = src + (r < rows ? r : rows - 1) * cols;
    // every load is made, whole (one that hangs over the row's end is moved back to end with it)
    auto const load = [&](unsigned t) {
      size_t const c = static_cast<size_t>(t) * 64 + c8;
      return *reinterpret_cast<CeOct<T> const *>(row + (c + 8 <= cols ? c : cols - 8));
    };
    CeOct<T> keep[KEEP];
    float m = 0.0f;
    if (narrow) {
      for (size_t c = 0; c < cols; ++c) m = ce_finite_max(m, static_cast<float>(row[c]));
    } else if (kept) {
#pragma unroll
      for (int k = 0; k < KEEP; ++k) keep[k] = load(first + step * k < tiles ? first + step * k : 0);
#pragma unroll
      for (int k = 0; k < KEEP; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) m = ce_finite_max(m, static_cast<float>(keep[k].v[i]));
    } else {
#pragma unroll 4
      for (unsigned t = wave; t < tiles; t += 4) {
        CeOct<T> const o = load(t);
#pragma unroll
        for (int i = 0; i < 8; ++i) m = ce_finite_max(m, static_cast<float>(o.v[i]));
      }
    }
#pragma unroll
    for (int o = 1; o < 8; o *= 2) m = fmaxf(m, __shfl_xor(m, o));
    if constexpr (!ALONE) {
      if ((lane & 7) == 0) top[flip][wave][r8] = m;
      __syncthreads();
      m = fmaxf(fmaxf(top[flip][0][r8], top[flip][1][r8]), fmaxf(top[flip][2][r8], top[flip][3][r8]));
      flip ^= 1;
    }
    float const scale = ce_scale(m);
    // across = as * ratio, ratio = weight * scale_across / scale
    // (a row of zeros has no share in a product, so none in the largest either)
    float ratio = r < rows ? 1.0f : 0.0f, un = m > 0.0f ? ce_unscale(scale) : 0.0f, s2 = scale;
    if ((lane & 7) == 0 && (ALONE || wave == 0)) unscale[r] = un;
    if constexpr (LABELS) {
      int const l = r < rows ? a.labels[r] : -1;
      float const w = l >= 0 && static_cast<size_t>(l) < a.V ? ce_row_weight(a, r) : 0.0f;
      s2 = ce_scale(fabsf(w) * m);
      ratio = l >= 0 && static_cast<size_t>(l) < a.V ? w * (s2 * ce_unscale(scale)) : 0.0f;
      un = fabsf(w) * m > 0.0f ? ce_unscale(s2) : 0.0f;
      if ((lane & 7) == 0 && (ALONE || wave == 0)) unscale_across[r] = un;
    }
    mine = fmaxf(mine, r < rows ? un : 0.0f);
    finest = fmaxf(finest, r < rows && un > 0.0f ? s2 : 0.0f);
    auto const pack = [&](float const (&v)[8], char *dst) {
      half8 hi, lo;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float y = v[i];
        if constexpr (NP == 2) asm("" : "+v"(y));  // (one value for both planes)
        _Float16 const h = static_cast<_Float16>(y);
        hi[i] = h;
        if constexpr (NP == 2) lo[i] = static_cast<_Float16>(y - static_cast<float>(h));
      }
      *reinterpret_cast<half8 *>(dst) = hi;
      if constexpr (NP == 2) *reinterpret_cast<half8 *>(dst + kFragBytes) = lo;
    };
    auto const tile = [&](unsigned t, CeOct<T> const &o) {
      float x[8];
      size_t const c = static_cast<size_t>(t) * 64 + c8;
      if (narrow) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = r < rows && c + i < cols ? static_cast<float>(row[c + i < cols ? c + i : cols - 1]) * scale : 0.0f;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = r < rows && c + 8 <= cols ? static_cast<float>(o.v[i]) * scale : 0.0f;
        if (c < cols && c + 8 > cols && r < rows) {  // the row's end: the octet was moved back by c + 8 - cols
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c + i < cols) x[i] = static_cast<float>(row[c + i]) * scale;
        }
      }
      if (as != nullptr) {
        size_t const frag = (r / 32) * kblocks_as + t * 4 + (lane & 7) / 2;
        pack(x, as + frag * NP * kFragBytes + ((lane & 1) * 32 + (r & 31)) * 16);
      }
      if (across != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) turn[wave][r8][c8 + i] = !LABELS || ratio != 0.0f ? x[i] * (LABELS ? ratio : 1.0f) : 0.0f;
        __builtin_amdgcn_wave_barrier();
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = turn[wave][i][lane];
        __builtin_amdgcn_wave_barrier();
        size_t const f = static_cast<size_t>(t) * 64 + lane;
        size_t const frag = (f / 32) * kblocks_across + r0 / 16;
        pack(y, across + frag * NP * kFragBytes + ((r0 / 8 & 1) * 32 + (f & 31)) * 16);
      }
    };
    if (kept) {
#pragma unroll
      for (int k = 0; k < KEEP; ++k)
        if (first + step * k < tiles) tile(first + step * k, keep[k]);
    } else {
#pragma unroll 2
      for (unsigned t = wave; t < tiles; t += 4) tile(t, narrow ? CeOct<T>{} : load(t));
    }
  }
  if (most.w == nullptr) return;
  mine = ce_wave_max(mine);
  finest = ce_wave_max(finest);
  if constexpr (ALONE) {  // (otherwise the wavefronts have seen the same rows)
    if (lane == 0) {
      top[0][wave][0] = mine;
      top[0][wave][1] = finest;
    }
    __syncthreads();
    mine = fmaxf(fmaxf(top[0][0][0], top[0][1][0]), fmaxf(top[0][2][0], top[0][3][0]));
    finest = fmaxf(fmaxf(top[0][0][1], top[0][1][1]), fmaxf(top[0][2][1], top[0][3][1]));
  }
  if constexpr (LABELS) {
    if (threadIdx.x == 0) {
      most.parts[blockIdx.x] = mine;
      most.parts[most.nparts + blockIdx.x] = finest;
    }
    if (blockIdx.x == 0)
      for (unsigned q = threadIdx.x; q < 2 * most.pieces; q += kCeBlock) most.w[q] = 0.0f;
  } else {
    if (threadIdx.x < 2) {
      // (powers of two, mostly the same ones: who finds at least its own there, however old the value, has nothing to add)
      unsigned *const to = reinterpret_cast<unsigned *>(most.w) + threadIdx.x * most.pieces + most.piece;
      unsigned const x = __float_as_uint(threadIdx.x == 0 ? mine : finest);
      if (__hip_atomic_load(to, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) < x) atomicMax(to, x);
    }
    if (most.piece == 0 && blockIdx.x == 0 && wave < 2) {
      float const x = ce_largest(most.parts + wave * most.nparts, most.nparts, lane);
      if (lane == 0) most.x[wave] = x;
    }
  }
}

// Tile number -> (ti, tj) in bands of 8 ti: the tiles that run together on an XCD share operand rows.
__device__ __forceinline__ void ce_tile(unsigned id, unsigned ni, unsigned nj, unsigned &ti, unsigned &tj) {
  unsigned const band = id / (8 * nj), left = ni - band * 8, w = left < 8 ? left : 8, r = id - band * 8 * nj;
  tj = r / w;
  ti = band * 8 + r - tj * w;
}

// What a sum of exponentials around m counts in one around `most` >= m.  Nothing has been summed around -infinity (or NaN,
// which times zero stays NaN).
__device__ __forceinline__ float ce_join_factor(float m, float most) { return m > -INFINITY ? __expf(m - most) : 0.0f; }

// The logits of a tile: classes i of the piece (P = W packed), rows j of the batch (Q = X packed).
struct CeLogits {
  char const *P, *Q;
  float const *unscale_x, *unscale_w;  // of the rows of the batch, of the piece's classes
  // backward: what undoes the scale of X's rows times dloss; the largest of those and their largest scale, both of unscale_w
  float const *unscale_xw, *most_x, *finest_x, *most_w, *finest_w;
  float *dl;                           // dL [padded rows][dl_stride] in fp32, where the factors lie far apart
  size_t dl_stride;
  unsigned ni, nj, kblocks, stages;    // kblocks: of a row block in memory
  size_t v0, vn;                     // first class of the piece, classes in it
};

// The biases of a lane's 16 classes of a 32-class block from c0 on; -infinity beyond the piece, which makes the logit that.
// (Every load is made, of the last class at most: loads behind conditions of their own would each be waited for.)
__device__ __forceinline__ f32x16 ce_biases(CeArgs const &a, CeLogits const &g, size_t c0, int lane) {
  f32x16 v = {};
  size_t const c1 = c0 + 4 * (lane >> 5);
  if (a.bias != nullptr) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      size_t const c = c1 + 8 * (r >> 2) + (r & 3);
      v[r] = a.bias[g.v0 + (c < g.vn ? c : g.vn - 1)];
    }
  }
  if (c0 + 32 > g.vn) {
#pragma unroll
    for (int r = 0; r < 16; ++r) v[r] = c1 + 8 * (r >> 2) + (r & 3) < g.vn ? v[r] : -INFINITY;
  }
  return v;
}

// What undoes the scale of those classes (padding has entries too).
__device__ __forceinline__ f32x16 ce_unscales(CeLogits const &g, size_t c0, int lane) {
  f32x16 v;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    f32x4 const x = *reinterpret_cast<f32x4 const *>(g.unscale_w + c0 + 4 * (lane >> 5) + 8 * q);
#pragma unroll
    for (int t = 0; t < 4; ++t) v[q * 4 + t] = x[t];
  }
  return v;
}

// Bound by the matrix pipe: 229 us for [8192 x 2048] x [8192 x 2048] BF16 = 1200 TFLOP/s, 142 us for [777 x 1000] FP32 against
// 30011 classes (985 TFLOP/s of 16-bit products); the same product without an epilogue takes 216 us.
// part[half tile of classes][Bp] = (max, sum of exp(z - max)); target[b] = the label's logit.
template <int T, int NP>
__global__ __launch_bounds__(256, T >= 256 ? 1 : 2) void k_ce_stats(CeArgs a, CeLogits g, float2 *part, size_t part_stride, size_t part_row0,
                                                                   float *target) {
  using H = HalfTile<T, T, NP>;
  unsigned ti, tj;
  ce_tile(xcd_consecutive(blockIdx.x, gridDim.x), g.ni, g.nj, ti, tj);
  size_t const rs = static_cast<size_t>(g.kblocks) * NP * kFragBytes;
  HalfAcc<H> acc;
  half_gemm<H>(acc, g.P + ti * (T / 32) * rs, g.Q + tj * (T / 32) * rs, rs, rs, g.stages);
  int const lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  size_t const c0 = static_cast<size_t>(ti) * T + (wave >> 1) * (T / 2);
  size_t const b0 = static_cast<size_t>(tj) * T + (wave & 1) * (T / 2) + (lane & 31);
  float ux[H::kNB];
#pragma unroll
  for (int n = 0; n < H::kNB; ++n) ux[n] = g.unscale_x[b0 + n * 32 < a.B ? b0 + n * 32 : a.B - 1];
#pragma unroll
  for (int m = 0; m < H::kMB; ++m) {
    f32x16 const bias = ce_biases(a, g, c0 + m * 32, lane), uw = ce_unscales(g, c0 + m * 32, lane);
#pragma unroll
    for (int n = 0; n < H::kNB; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc.v[m][n][r] = acc.v[m][n][r] * ux[n] * uw[r] + bias[r];
  }
#pragma unroll
  for (int n = 0; n < H::kNB; ++n) {
    size_t const b = b0 + n * 32;
    bool const in = b < a.B;
    float top = -INFINITY;
#pragma unroll
    for (int m = 0; m < H::kMB; ++m)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, acc.v[m][n][r]);
    float sum = 0.0f;
    float const base = top > -INFINITY ? top : 0.0f;
#pragma unroll
    for (int m = 0; m < H::kMB; ++m)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum += __expf(acc.v[m][n][r] - base);
    // the label's class, where it lies in this wavefront's rows
    long long const at = in ? static_cast<long long>(a.labels[b]) - static_cast<long long>(g.v0 + c0) : -1;
    if (__any(at >= 0 && at < T / 2)) {
#pragma unroll
      for (int m = 0; m < H::kMB; ++m)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (at == m * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3) && static_cast<size_t>(at) + c0 < g.vn) target[b] = acc.v[m][n][r];
    }
    float const top2 = __shfl_xor(top, 32), sum2 = __shfl_xor(sum, 32);
    float const most = fmaxf(top, top2);
    sum = sum * ce_join_factor(top, most) + sum2 * ce_join_factor(top2, most);
    if (lane < 32 && in) part[(part_row0 + ti * 2 + (wave >> 1)) * part_stride + b] = make_float2(most, sum);
  }
}

// kRows rows of the batch per workgroup: 1024 / kRows threads each join every so manieth partial, eight of them on their way
// at a time, then one another's, in a fixed order.  8192 rows of 512 partials: 8.6 us; 120 rows of 1508: 7.6 (34 with 64 rows a
// workgroup).
template <int kRows>
__global__ __launch_bounds__(1024) void k_ce_join(CeArgs a, float2 const *part, size_t part_stride, size_t parts, float const *target) {
  constexpr int kParts = 1024 / kRows;
  __shared__ float2 lds[kParts][kRows];
  size_t const b = static_cast<size_t>(blockIdx.x) * kRows + threadIdx.x % kRows, in = b < a.B ? b : a.B - 1;
  int const w = threadIdx.x / kRows;
  float2 s = make_float2(-INFINITY, 0.0f);
  auto const join = [&](float2 p) {
    float const most = fmaxf(s.x, p.x);
    s.y = s.y * ce_join_factor(s.x, most) + p.y * ce_join_factor(p.x, most);
    s.x = most;
  };
  size_t p = w;
  for (; p + 7 * kParts < parts; p += 8 * kParts) {
    float2 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = part[(p + i * kParts) * part_stride + in];
#pragma unroll
    for (int i = 0; i < 8; ++i) join(v[i]);
  }
  for (; p < parts; p += kParts) join(part[p * part_stride + in]);
  lds[w][threadIdx.x % kRows] = s;
  __syncthreads();
  for (int o = kParts / 2; o > 0; o >>= 1) {
    if (w < o) {
      join(lds[w + o][threadIdx.x % kRows]);
      lds[w][threadIdx.x % kRows] = s;
    }
    __syncthreads();
  }
  if (w != 0 || b >= a.B) return;
  float const lse = s.x + logf(s.y);
  a.lse[b] = lse;
  int const l = a.labels[b];
  a.loss[b] = l >= 0 && static_cast<size_t>(l) < a.V ? lse - target[b] : 0.0f;
}

// ---- few rows: W is read once, as it lies ---------------------------------------------------------------------------
// Forward for up to 64 rows of the batch (NB blocks of 32), bound by reading W: packing it would move it three times.  A
// workgroup takes 32 VB classes at a time; its NW wavefronts share the features between them (every NW-th 64 bytes of a
// lane's row), multiply the tensors' own type (bf16, or fp32 on the fp32 matrix pipe, which keeps up with memory at 64 rows) and
// join in LDS.  The last workgroup to finish joins all partial sums, in a fixed order.  [24 x 2048] BF16 against 65536
// classes: 55 us = 4.9 TB/s; [4 x 512] FP32 against 10007: 14 us, the latency of loads, two barriers and the joining.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// A lane's 64 bytes of a step: four pieces of 16, 16 G apart (G lanes share a row, so that a load takes 16 G consecutive
// bytes of it); at any alignment.
struct CeLine {
  u32x4 q[4];
};
template <class E>
struct __attribute__((packed, aligned(sizeof(E)))) CePiece {
  u32x4 q;
};

template <class E, int G>
__device__ __forceinline__ CeLine ce_line(E const *p) {
  CeLine r;
#pragma unroll
  for (int t = 0; t < 4; ++t) r.q[t] = reinterpret_cast<CePiece<E> const *>(p + t * (G * 16 / static_cast<int>(sizeof(E))))->q;
  return r;
}
// The same where the row ends at K; what lies beyond counts as zero.  Of bf16 rows a piece over the end is loaded from where it
// ends with the row and shifted down (16 loads of 2 bytes instead: 22.4 us, not 19.8, for [16 x 1020] against 21246 classes);
// of fp32 rows the values are loaded one by one (shifted: 57 us, not 50, for [55 x 101] against 114534).
template <class E, int G>
__device__ __forceinline__ CeLine ce_line_tail(E const *row, size_t k, size_t K) {
  constexpr int N = 16 / sizeof(E);
  if (sizeof(E) == 4 || K < N) {
    union {
      E e[4 * N];
      CeLine l;
    } u;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < N; ++i) u.e[t * N + i] = k + t * G * N + i < K ? row[k + t * G * N + i] : static_cast<E>(0.0f);
    return u.l;
  }
  CeLine r;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    size_t const at = k + t * G * N, from = at + N <= K ? at : K - N;
    r.q[t] = reinterpret_cast<CePiece<E> const *>(row + from)->q;
  }
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    size_t const at = k + t * G * N, over = at + N <= K ? 0 : at + N - K;
    unsigned __int128 const v = __builtin_bit_cast(unsigned __int128, r.q[t]);
    r.q[t] = __builtin_bit_cast(u32x4, over < N ? v >> (static_cast<unsigned>(over) * 8 * static_cast<unsigned>(sizeof(E))) : 0);
  }
  return r;
}

// Blocks of RB classes x RB rows of the batch: RB = 32 or, for up to 16 rows of the batch, 16 (fp32 products of 32 columns
// cost 3.5 us where four rows of the batch wait for 20 MB).  A lane holds class lane % RB, and piece lane / RB of every G =
// 64 / RB of its row; its results are column lane % RB.
template <int RB>
struct CeShape;
template <>
struct CeShape<32> {
  using Acc = f32x16;
  static constexpr int kRegs = 16;
  static __device__ __forceinline__ int row(int r, int lane) { return 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3); }
  static __device__ __forceinline__ Acc mul(bf16x8 w, bf16x8 x, Acc acc) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(w, x, acc, 0, 0, 0); }
  static __device__ __forceinline__ Acc mul(float w, float x, Acc acc) { return __builtin_amdgcn_mfma_f32_32x32x2f32(w, x, acc, 0, 0, 0); }
};
template <>
struct CeShape<16> {
  using Acc = f32x4;
  static constexpr int kRegs = 4;
  static __device__ __forceinline__ int row(int r, int lane) { return 4 * (lane >> 4) + r; }
  static __device__ __forceinline__ Acc mul(bf16x8 w, bf16x8 x, Acc acc) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x, acc, 0, 0, 0); }
  static __device__ __forceinline__ Acc mul(float w, float x, Acc acc) { return __builtin_amdgcn_mfma_f32_16x16x4f32(w, x, acc, 0, 0, 0); }
};

template <class E, int RB>
__device__ __forceinline__ typename CeShape<RB>::Acc ce_line_mfma(CeLine const &w, CeLine const &x, typename CeShape<RB>::Acc acc) {
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if constexpr (sizeof(E) == 2) {
      acc = CeShape<RB>::mul(__builtin_bit_cast(bf16x8, w.q[t]), __builtin_bit_cast(bf16x8, x.q[t]), acc);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) acc = CeShape<RB>::mul(__uint_as_float(w.q[t][i]), __uint_as_float(x.q[t][i]), acc);
    }
  }
  return acc;
}

template <class E, int RB, int VB, int NB, int NW>
__global__ __launch_bounds__(NW * 64, 2) void k_ce_direct(CeArgs a, float2 *part, float *target, unsigned *ticket) {
  using S = CeShape<RB>;
  constexpr int N = 64 / sizeof(E), G = 64 / RB;   // features of a line; lines of a row in a step
  constexpr int kShare = VB * S::kRegs / NW;        // registers of a wavefront's share of the results
  __shared__ float red[NW][NB][VB * S::kRegs][64];
  __shared__ float2 sums[NW][NB * RB];
  __shared__ float hit[NB * RB];
  __shared__ int last;
  int const lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  E const *w[VB], *x[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    size_t const b = static_cast<size_t>(n * RB + lane % RB);
    x[n] = static_cast<E const *>(a.X) + (b < a.B ? b : a.B - 1) * a.K;
  }
  auto const rows = [&](size_t v0) {
#pragma unroll
    for (int m = 0; m < VB; ++m) {
      size_t const v = v0 + m * RB + lane % RB;
      w[m] = static_cast<E const *>(a.W) + (v < a.V ? v : a.V - 1) * a.K;
    }
  };
  // G lines of every row are a step; the wavefront's next step is on its way meanwhile, also
  // across blocks of classes
  size_t const steps = a.K / (G * N), mine = static_cast<size_t>(lane / RB) * (N / 4);
  bool const tail = a.K % (G * N) != 0 && static_cast<int>(steps % NW) == wave;
  CeLine lw[VB], lx[NB];
  auto const load = [&](size_t s) {
#pragma unroll
    for (int m = 0; m < VB; ++m) lw[m] = ce_line<E, G>(w[m] + s * G * N + mine);
#pragma unroll
    for (int n = 0; n < NB; ++n) lx[n] = ce_line<E, G>(x[n] + s * G * N + mine);
  };
  auto const join = [](float2 &p, float2 q) {
    float const most = fmaxf(p.x, q.x);
    p.y = p.y * ce_join_factor(p.x, most) + q.y * ce_join_factor(q.x, most);
    p.x = most;
  };
  float2 mine_sum = make_float2(-INFINITY, 0.0f);  // of row `lane`, in the first wavefront
  size_t const stride = static_cast<size_t>(gridDim.x) * (RB * VB);
  size_t v0 = static_cast<size_t>(blockIdx.x) * (RB * VB);
  rows(v0);
  if (static_cast<size_t>(wave) < steps) load(wave);
  for (; v0 < a.V; v0 += stride) {
    typename S::Acc acc[VB][NB];
#pragma unroll
    for (int m = 0; m < VB; ++m)
#pragma unroll
      for (int n = 0; n < NB; ++n) acc[m][n] = typename S::Acc{};
    auto const multiply = [&](CeLine const (&cw)[VB], CeLine const (&cx)[NB]) {
#pragma unroll
      for (int m = 0; m < VB; ++m)
#pragma unroll
        for (int n = 0; n < NB; ++n) acc[m][n] = ce_line_mfma<E, RB>(cw[m], cx[n], acc[m][n]);
    };
    if (tail) {
      CeLine tw[VB], tx[NB];
#pragma unroll
      for (int m = 0; m < VB; ++m) tw[m] = ce_line_tail<E, G>(w[m], steps * G * N + mine, a.K);
#pragma unroll
      for (int n = 0; n < NB; ++n) tx[n] = ce_line_tail<E, G>(x[n], steps * G * N + mine, a.K);
      multiply(tw, tx);
    }
    CeLine cw[VB], cx[NB];
    size_t s = wave;
    for (; s + NW < steps; s += NW) {
#pragma unroll
      for (int m = 0; m < VB; ++m) cw[m] = lw[m];
#pragma unroll
      for (int n = 0; n < NB; ++n) cx[n] = lx[n];
      load(s + NW);
      multiply(cw, cx);
    }
    if (s < steps) {
#pragma unroll
      for (int m = 0; m < VB; ++m) cw[m] = lw[m];
#pragma unroll
      for (int n = 0; n < NB; ++n) cx[n] = lx[n];
      if (v0 + stride < a.V) {
        rows(v0 + stride);
        load(wave);
      }
      multiply(cw, cx);
    } else if (v0 + stride < a.V) {
      rows(v0 + stride);
    }
#pragma unroll
    for (int m = 0; m < VB; ++m)
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int r = 0; r < S::kRegs; ++r) red[wave][n][m * S::kRegs + r][lane] = acc[m][n][r];
    __syncthreads();
    // a wavefront finishes its share of the results' registers
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      size_t const b = static_cast<size_t>(n * RB + lane % RB);
      long long const at = b < a.B ? static_cast<long long>(a.labels[b]) - static_cast<long long>(v0) : -1;
      float z[kShare];
      float top = -INFINITY;
#pragma unroll
      for (int t = 0; t < kShare; ++t) {
        int const reg = wave * kShare + t, c = reg / S::kRegs * RB + S::row(reg % S::kRegs, lane);
        float s1 = 0.0f;
#pragma unroll
        for (int q = 0; q < NW; ++q) s1 += red[q][n][reg][lane];
        if (v0 + c < a.V) {
          if (a.bias != nullptr) s1 += a.bias[v0 + c];
          if (at == c) hit[n * RB + lane % RB] = s1;
        } else {
          s1 = -INFINITY;
        }
        z[t] = s1;
        top = fmaxf(top, s1);
      }
      float const base = top > -INFINITY ? top : 0.0f;
      float sum = 0.0f;
#pragma unroll
      for (int t = 0; t < kShare; ++t) sum += __expf(z[t] - base);
#pragma unroll
      for (int o = RB; o < 64; o *= 2) {
        float const top2 = __shfl_xor(top, o), sum2 = __shfl_xor(sum, o), most = fmaxf(top, top2);
        sum = sum * ce_join_factor(top, most) + sum2 * ce_join_factor(top2, most);
        top = most;
      }
      float const most = top;
      if (lane < RB) sums[wave][n * RB + lane] = make_float2(most, sum);
    }
    __syncthreads();
    // (the next block's sums are written behind its own first barrier, which the first wavefront reaches after this)
    if (wave == 0 && lane < NB * RB && static_cast<size_t>(lane) < a.B) {
#pragma unroll
      for (int q = 0; q < NW; ++q) join(mine_sum, sums[q][lane]);
      long long const at = static_cast<long long>(a.labels[lane]) - static_cast<long long>(v0);
      if (at >= 0 && at < RB * VB && v0 + at < a.V) __hip_atomic_store(&target[lane], hit[lane], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  // The first wavefront alone writes what other workgroups read, past the caches (device scope), waits until that is done
  // and takes a ticket; who draws the last one reads it all, past the caches as well.  A release and acquire instead would
  // write back and empty the L2 for every workgroup.
  if (wave == 0) {
    if (lane < NB * RB && static_cast<size_t>(lane) < a.B)
      __hip_atomic_store(reinterpret_cast<unsigned long long *>(part + static_cast<size_t>(blockIdx.x) * a.B + lane),
                         static_cast<unsigned long long>(__float_as_uint(mine_sum.y)) << 32 | __float_as_uint(mine_sum.x), __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0);
    asm volatile("" ::: "memory");
    if (lane == 0) {
      unsigned const t = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      last = t + 1 == gridDim.x;
      if (last) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  __syncthreads();
  if (!last) return;
  // a power of two of threads side by side over the rows of the batch, the others share the partials
  int wide = 1;
  while (wide < static_cast<int>(a.B)) wide *= 2;
  int const slices = NW * 64 / wide, b = static_cast<int>(threadIdx.x) & (wide - 1), slice = static_cast<int>(threadIdx.x) / wide;
  float2 *const tree = reinterpret_cast<float2 *>(&red[0][0][0][0]);
  float2 p = make_float2(-INFINITY, 0.0f);
  int label = -1;
  float chosen = 0.0f;
  if (static_cast<size_t>(b) < a.B) {
    label = a.labels[b];
    if (label >= 0 && static_cast<size_t>(label) < a.V) chosen = __hip_atomic_load(&target[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    auto const at = [&](unsigned q) {
      unsigned long long const o =
          __hip_atomic_load(reinterpret_cast<unsigned long long *>(part + static_cast<size_t>(q) * a.B + b), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      return make_float2(__uint_as_float(static_cast<unsigned>(o)), __uint_as_float(static_cast<unsigned>(o >> 32)));
    };
    unsigned q = slice;
    for (; q + 15 * slices < gridDim.x; q += 16 * slices) {
      float2 o[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i] = at(q + i * slices);
#pragma unroll
      for (int i = 0; i < 16; ++i) join(p, o[i]);
    }
    for (; q < gridDim.x; q += slices) join(p, at(q));
  }
  tree[threadIdx.x] = p;
  __syncthreads();
  for (int o = slices / 2; o > 0; o >>= 1) {
    if (slice < o) {
      join(p, tree[threadIdx.x + o * wide]);
      tree[threadIdx.x] = p;
    }
    __syncthreads();
  }
  if (slice != 0 || static_cast<size_t>(b) >= a.B) return;
  float const lse = p.x + logf(p.y);
  a.lse[b] = lse;
  a.loss[b] = label >= 0 && static_cast<size_t>(label) < a.V ? lse - chosen : 0.0f;
}

// The sums over the 32 lanes of a half wavefront of its 16 values each, scattered: lanes halve what they hold with a partner
// (16, 8 and 4 lanes away, then in mirrored fours) until one value is left, which the neighbour shares.  Value
// ce_scatter_row(lane) ends up in the lane.
template <int CTRL>
__device__ __forceinline__ float ce_dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ int ce_scatter_row(int lane) { return (lane >> 4 & 1) * 8 + (lane >> 3 & 1) * 4 + (lane >> 2 & 1) * 2 + (lane >> 1 & 1); }
__device__ __forceinline__ float ce_scatter_sum(f32x16 const &v, int lane) {
  float a[8], b[4], c[2];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    unsigned const lo = __float_as_uint(v[i]), hi = __float_as_uint(v[i + 8]);
    // rows of 16 lanes: the even one keeps the low values of both, the odd one the high
    auto const x = __builtin_amdgcn_permlane16_swap(lo, hi, false, false);
    a[i] = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  }
  bool const up8 = lane & 8, up4 = lane & 4, up2 = lane & 2;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float const keep = up8 ? a[i + 4] : a[i], give = up8 ? a[i] : a[i + 4];
    b[i] = keep + ce_dpp<0x128>(give);  // lane ^ 8: rotated by 8 in 16
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float const keep = up4 ? b[i + 2] : b[i], give = up4 ? b[i] : b[i + 2];
    // lane ^ 4: mirrored in 8 (lane ^ 7), then in 4 (lane ^ 3)
    c[i] = keep + ce_dpp<0x1B>(ce_dpp<0x141>(give));
  }
  float const keep = up2 ? c[1] : c[0], give = up2 ? c[0] : c[1];
  float const d = keep + ce_dpp<0x4E>(give);  // lane ^ 2
  return d + ce_dpp<0xB1>(d);                 // lane ^ 1
}

// dL of a tile, packed for dX (rows of the batch, k = classes; times what undoes the scale of W's row, as a share of the
// piece's largest) and for dW (rows are classes, k = rows of the batch; times what undoes the scale of X's row, as a share of
// the largest): the factors of the products' k that do not come out of their sums, powers of two, so that the planes are
// rounded once and multiplied in f16 (a share of 2^-s costs an element s of the bits above 2^-40).  Bound by the matrix pipe and by
// writing both packings: 300 - 310 us for a piece of 8192 classes, [8192 x 2048] BF16, 175 - 200 us for [777 x 1000] FP32 against
// 30011.  DB: also the sums of dloss dL over each half tile of rows.
// FAR: dL in fp32 instead.
template <int T, int NP, bool DB, bool FAR>
__device__ __forceinline__ void ce_grad_tile(CeArgs const &a, CeLogits const &g, char *dlb, char *dlv, unsigned kblocks_v, unsigned kblocks_b,
                                             float *dbpart, size_t dbpart_stride) {
  using H = HalfTile<T, T, NP>;
  unsigned ti, tj;
  ce_tile(xcd_consecutive(blockIdx.x, gridDim.x), g.ni, g.nj, ti, tj);
  size_t const rs = static_cast<size_t>(g.kblocks) * NP * kFragBytes;
  HalfAcc<H> acc;
  half_gemm<H>(acc, g.P + ti * (T / 32) * rs, g.Q + tj * (T / 32) * rs, rs, rs, g.stages);
  int const lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  half8 const id0 = half_identity(0, lane), id1 = half_identity(1, lane);
  // (powers of two, so their inverses are exact)
  float const most_w = g.most_w[0], most_x = g.most_x[0];
  float const inv_w = most_w > 0.0f ? 1.0f / most_w : 0.0f, inv_x = most_x > 0.0f ? 1.0f / most_x : 0.0f;
  size_t const c0 = static_cast<size_t>(ti) * T + (wave >> 1) * (T / 2);
  size_t const b0 = static_cast<size_t>(tj) * T + (wave & 1) * (T / 2);
  size_t const rb = static_cast<size_t>(kblocks_v) * NP * kFragBytes, rv = static_cast<size_t>(kblocks_b) * NP * kFragBytes;
  // of this lane's rows of the batch: unscale, lse, weight, share of the largest, and the label's class from c0 on (-1: none here)
  float ux[H::kNB], lse[H::kNB], weight[H::kNB];
  _Float16 fx[H::kNB];
  int at[H::kNB];
  bool live[H::kNB];
#pragma unroll
  for (int n = 0; n < H::kNB; ++n) {
    size_t const b = b0 + n * 32 + (lane & 31), in = b < a.B ? b : a.B - 1;
    int const label = a.labels[in];
    ux[n] = g.unscale_x[in];
    lse[n] = a.lse_in[in];
    weight[n] = a.dloss != nullptr ? a.dloss[in] : 1.0f;
    fx[n] = static_cast<_Float16>(g.unscale_xw[in] * inv_x);
    live[n] = b < a.B && label >= 0 && static_cast<size_t>(label) < a.V;
    long long const c = static_cast<long long>(label) - static_cast<long long>(g.v0 + c0);
    at[n] = live[n] && c >= 0 && c < T / 2 ? static_cast<int>(c) : -1;
  }
#pragma unroll
  for (int m = 0; m < H::kMB; ++m) {
    f32x16 const bias = ce_biases(a, g, c0 + m * 32, lane), uw = ce_unscales(g, c0 + m * 32, lane);
    half4 fw[4];
#pragma unroll
    for (int r = 0; r < 16; ++r) fw[r >> 2][r & 3] = static_cast<_Float16>(uw[r] * inv_w);
    f32x16 sum = {};
    bool const whole = c0 + m * 32 + 32 <= g.vn;
#pragma unroll
    for (int n = 0; n < H::kNB; ++n) {
      f32x16 z = acc.v[m][n];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        int const c = m * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
        float p = __expf(z[r] * ux[n] * uw[r] + bias[r] - lse[n]);
        // (the forward may have rounded z otherwise: beyond some 10^5 that is more than 1, and e^1 times 2^15 overflows f16; a NaN stays)
        p = p > 1.0f ? 1.0f : p;
        p -= at[n] == c ? 1.0f : 0.0f;
        // (a class beyond the piece: its logit is -infinity, but a row's lse may be too)
        z[r] = live[n] && (whole || c0 + c < g.vn) ? p : 0.0f;
        if constexpr (DB) sum[r] += live[n] ? weight[n] * z[r] : 0.0f;
      }
      size_t const ib = c0 / 32 + m, jb = b0 / 32 + n;
      if constexpr (FAR) {
        float *const to = g.dl + (b0 + n * 32 + (lane & 31)) * g.dl_stride + c0 + m * 32 + 4 * (lane >> 5);
#pragma unroll
        for (int k = 0; k < 4; ++k) *reinterpret_cast<f32x4 *>(to + 8 * k) = f32x4{z[k * 4], z[k * 4 + 1], z[k * 4 + 2], z[k * 4 + 3]};
        continue;
      }
      HalfQuads<NP> const q = half_planes<NP>(z * kCeDl);
      HalfQuads<NP> qb, qv;
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          qb.h[p][k] = q.h[p][k] * fw[k];
          qv.h[p][k] = q.h[p][k] * fx[n];
        }
      half_store<NP>(dlb + jb * rb + ib * 2 * NP * kFragBytes, half_joined<NP>(qb), lane);
      half_store<NP>(dlv + ib * rv + jb * 2 * NP * kFragBytes, half_flip<NP>(half_joined<NP>(qv), id0, id1), lane);
    }
    if constexpr (DB) {
      float const s = ce_scatter_sum(sum, lane);
      int const r = ce_scatter_row(lane);
      if ((lane & 1) == 0)
        dbpart[(tj * 2 + (wave & 1)) * dbpart_stride + c0 + m * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)] = s;
    }
  }
}

__device__ __forceinline__ bool ce_far(CeLogits const &g) { return ce_apart(g.most_w, g.finest_w) || ce_apart(g.most_x, g.finest_x); }

template <int T, int NP, bool DB>
__global__ __launch_bounds__(256, T >= 256 ? 1 : 2) void k_ce_grad(CeArgs a, CeLogits g, char *dlb, char *dlv, unsigned kblocks_v,
                                                                  unsigned kblocks_b, float *dbpart, size_t dbpart_stride) {
  // (chosen before the K loop: with both epilogues behind one, neither has the registers it needs, 319 -> 339 us)
  if (ce_far(g))
    ce_grad_tile<T, NP, DB, true>(a, g, dlb, dlv, kblocks_v, kblocks_b, dbpart, dbpart_stride);
  else
    ce_grad_tile<T, NP, DB, false>(a, g, dlb, dlv, kblocks_v, kblocks_b, dbpart, dbpart_stride);
}

static __global__ __launch_bounds__(kCeBlock) void k_ce_db(float const *part, size_t stride, unsigned parts, size_t n, float *db, float scale, int accumulate) {
  size_t const c = static_cast<size_t>(blockIdx.x) * kCeBlock + threadIdx.x;
  if (c >= n) return;
  float s = 0.0f;
  for (unsigned p = 0; p < parts; ++p) s += part[p * stride + c];
  s *= scale;
  db[c] = accumulate ? db[c] + s : s;
}

// A 32 x 32 block of a product into row-major out [rows][cols] at (i0, j0), times `factor`, added to what is there or not.
// (A block inside has no conditions between its loads, which would each be waited for.)
template <class O>
__device__ __forceinline__ void ce_block_out(f32x16 const &v, float factor, O *out, size_t i0, size_t j0, size_t rows, size_t cols, bool add,
                                             int lane) {
  size_t const j = j0 + (lane & 31), i = i0 + 4 * (lane >> 5);
  if (i0 + 32 <= rows && j0 + 32 <= cols) {
    O *const p = out + i * cols + j;
    f32x16 w = {};
    if (add) {
#pragma unroll
      for (int r = 0; r < 16; ++r) w[r] = static_cast<float>(p[(8 * (r >> 2) + (r & 3)) * cols]);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) p[(8 * (r >> 2) + (r & 3)) * cols] = static_cast<O>(w[r] + v[r] * factor);
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      size_t const at = i + 8 * (r >> 2) + (r & 3);
      if (at < rows && j < cols) {
        O *const p = out + at * cols + j;
        *p = static_cast<O>((add ? static_cast<float>(*p) : 0.0f) + v[r] * factor);
      }
    }
  }
}

// A wavefront's blocks of a product on the fp32 matrix pipe over k = 0 .. count - 1, only where factors lie far apart: p(k, m),
// q(k, n) give four consecutive k from k on of this lane's row of block m and column of block n (zeros from count on), from the
// caches, eight k at a time and the next eight on their way.  A step takes two to three times as long with it: [777 x 1000] FP32
// against 30011 classes 1.82 ms instead of 0.74, [8192 x 2048] BF16 against 65536 14.3 instead of 8.2, [152 x 533] BF16 against
// 1838 167 us instead of 58.  Asking costs the other steps 0.3 - 0.6 us a launch: 0.4 - 2.4 %, and 2.5 us of that one's 55.
template <class H, class P, class Q>
__device__ __forceinline__ void ce_far_product(HalfAcc<H> &acc, size_t count, int lane, P &&p, Q &&q) {
  struct Eight {
    f32x4 x[H::kMB], y[H::kNB];
  };
  auto const load = [&](Eight &e, size_t k) {
#pragma unroll
    for (int m = 0; m < H::kMB; ++m) e.x[m] = p(k, m);
#pragma unroll
    for (int n = 0; n < H::kNB; ++n) e.y[n] = q(k, n);
  };
#pragma unroll
  for (int m = 0; m < H::kMB; ++m)
#pragma unroll
    for (int n = 0; n < H::kNB; ++n) acc.v[m][n] = f32x16{};
  Eight now, next;
  load(now, 4 * (lane >> 5));
  for (size_t k = 0; k < count; k += 8) {
    load(next, (k + 8 < count ? k + 8 : k) + 4 * (lane >> 5));
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int m = 0; m < H::kMB; ++m)
#pragma unroll
        for (int n = 0; n < H::kNB; ++n) acc.v[m][n] = __builtin_amdgcn_mfma_f32_32x32x2f32(now.x[m][t], now.y[n][t], acc.v[m][n], 0, 0, 0);
    now = next;
  }
}

// dW of a piece: classes i (P = dL packed by classes), features j (Q = dloss X packed by features), times `scale`.  216 - 228 us
// for 8192 classes, [8192 x 2048] BF16 = 1205 - 1270 TFLOP/s, falling with the clock in a long run.
template <int T, int NP, class O>
__global__ __launch_bounds__(256, T >= 256 ? 1 : 2) void k_ce_dw(CeArgs a, CeLogits g, char const *P, char const *Q, unsigned ni, unsigned nj,
                                                                unsigned kblocks, unsigned stages, float scale, O *out, size_t rows,
                                                                size_t cols, int accumulate) {
  using H = HalfTile<T, T, NP>;
  unsigned ti, tj;
  ce_tile(xcd_consecutive(blockIdx.x, gridDim.x), ni, nj, ti, tj);
  size_t const rs = static_cast<size_t>(kblocks) * NP * kFragBytes;
  int const lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float factor = g.most_x[0] * (scale * (1.0f / kCeDl));
  HalfAcc<H> acc;
  if (ce_far(g)) {
    size_t const i = static_cast<size_t>(ti) * T + (wave >> 1) * (T / 2) + (lane & 31), j = static_cast<size_t>(tj) * T + (wave & 1) * (T / 2) + (lane & 31);
    O const *const X = static_cast<O const *>(a.X);
    // (dL has whole tiles of rows, zero in padding and in rows left out, whose X may be anything)
    ce_far_product(
        acc, a.B, lane,
        [&](size_t b, int m) {
          float const *const d = g.dl + b * g.dl_stride + i + m * 32;
          return f32x4{d[0], d[g.dl_stride], d[2 * g.dl_stride], d[3 * g.dl_stride]};
        },
        [&](size_t b, int n) {
          size_t const f = j + n * 32 < cols ? j + n * 32 : cols - 1;
          f32x4 v;
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            size_t const in = b + t < a.B ? b + t : a.B - 1;
            int const l = a.labels[in];
            float const x = static_cast<float>(X[in * cols + f]), w = a.dloss != nullptr ? a.dloss[in] : 1.0f;
            v[t] = b + t < a.B && l >= 0 && static_cast<size_t>(l) < a.V && w != 0.0f ? w * x : 0.0f;
          }
          return v;
        });
    factor = scale;
  } else {
    half_gemm<H>(acc, P + ti * (T / 32) * rs, Q + tj * (T / 32) * rs, rs, rs, stages);
  }
#pragma unroll
  for (int m = 0; m < H::kMB; ++m)
#pragma unroll
    for (int n = 0; n < H::kNB; ++n)
      ce_block_out(acc.v[m][n], factor, out, static_cast<size_t>(ti) * T + (wave >> 1) * (T / 2) + m * 32,
                   static_cast<size_t>(tj) * T + (wave & 1) * (T / 2) + n * 32, rows, cols, accumulate != 0, lane);
}

// A slice of a piece's share of dX: rows of the batch i (P = dL packed by rows), features j (Q = W packed by features), summed
// over the piece's classes of the slice into out [slice][rows][cols]; the first piece writes, later ones add.  216 us for 8192
// classes, [8192 x 2048] BF16 = 1270 TFLOP/s; 228 - 239 where it adds.
template <int T, int NP, class E>
__global__ __launch_bounds__(256, T >= 256 ? 1 : 2) void k_ce_dx(CeLogits g, E const *W, char const *P, char const *Q, unsigned ni, unsigned nj,
                                                                unsigned kblocks, unsigned stages, unsigned per_slice, float *out,
                                                                size_t rows, size_t cols, int first) {
  using H = HalfTile<T, T, NP>;
  unsigned ti, tj;
  unsigned const id = xcd_consecutive(blockIdx.x, gridDim.x), slice = id / (ni * nj);
  ce_tile(id - slice * ni * nj, ni, nj, ti, tj);
  unsigned const s0 = slice * per_slice;
  if (s0 >= stages) return;  // a shorter last piece (the first has work for every slice)
  unsigned const count = stages - s0 < per_slice ? stages - s0 : per_slice;
  size_t const rs = static_cast<size_t>(kblocks) * NP * kFragBytes, skip = static_cast<size_t>(s0) * H::kStep;
  int const lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float factor = g.most_w[0] * (1.0f / kCeDl);
  HalfAcc<H> acc;
  if (ce_far(g)) {
    size_t const i = static_cast<size_t>(ti) * T + (wave >> 1) * (T / 2) + (lane & 31), j = static_cast<size_t>(tj) * T + (wave & 1) * (T / 2) + (lane & 31);
    size_t const c0 = static_cast<size_t>(s0) * H::KS * 16, left = g.vn > c0 ? g.vn - c0 : 0, most = static_cast<size_t>(count) * H::KS * 16;
    // (dL has whole tiles of classes, zero in padding; a slice is whole blocks of 16)
    ce_far_product(
        acc, left < most ? left : most, lane,
        [&](size_t c, int m) { return *reinterpret_cast<f32x4 const *>(g.dl + (i + m * 32) * g.dl_stride + c0 + c); },
        [&](size_t c, int n) {
          size_t const f = j + n * 32 < cols ? j + n * 32 : cols - 1;
          f32x4 v;
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            size_t const in = c0 + c + t;
            float const w = static_cast<float>(W[(in < g.vn ? in : g.vn - 1) * cols + f]);
            v[t] = in < g.vn ? w : 0.0f;
          }
          return v;
        });
    factor = 1.0f;
  } else {
    half_gemm<H>(acc, P + ti * (T / 32) * rs + skip, Q + tj * (T / 32) * rs + skip, rs, rs, count);
  }
  out += slice * rows * cols;
#pragma unroll
  for (int m = 0; m < H::kMB; ++m)
#pragma unroll
    for (int n = 0; n < H::kNB; ++n)
      ce_block_out(acc.v[m][n], factor, out, static_cast<size_t>(ti) * T + (wave >> 1) * (T / 2) + m * 32,
                   static_cast<size_t>(tj) * T + (wave & 1) * (T / 2) + n * 32, rows, cols, first == 0, lane);
}

// dX = scale dloss sum over slices, rows left out zero.  A workgroup per row and 1024 features.
template <class O>
__global__ __launch_bounds__(kCeBlock) void k_ce_dx_finish(CeArgs a, float const *acc, unsigned slices, O *dX) {
  size_t const b = blockIdx.x, k0 = static_cast<size_t>(blockIdx.y) * (kCeBlock * 4) + threadIdx.x;
  int const l = a.labels[b];
  bool const live = l >= 0 && static_cast<size_t>(l) < a.V;
  float const g = ce_row_weight(a, b) * a.scale;
  size_t const n = a.B * a.K;
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  size_t at[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) at[t] = b * a.K + (k0 + t * kCeBlock < a.K ? k0 + t * kCeBlock : a.K - 1);
  if (live) {
    for (unsigned q = 0; q < slices; ++q)
#pragma unroll
      for (int t = 0; t < 4; ++t) s[t] += acc[q * n + at[t]];
  }
#pragma unroll
  for (int t = 0; t < 4; ++t)
    if (k0 + t * kCeBlock < a.K) dX[at[t]] = static_cast<O>(live ? s[t] * g : 0.0f);
}

// ---- host ------------------------------------------------------------------------------------------------------------
struct CePlan {
  int T, Tw;                       // tile; of dW (not larger)
  size_t Bp, Kp, Vc, pieces;       // padded rows and features; classes of a piece (a multiple of T)
  unsigned slices, per_slice;      // of dX
  unsigned pack_x, pack_w;         // packing workgroups
  // offsets in the scratch
  size_t xp, xt, wp, wt, dlb, dlv, parts_x, unscale_x, unscale_xw, unscale_w, most_x, most_w, part, target, dxacc, dbpart, bytes;
};

// Packing workgroups for n (padded) rows: of 8 rows each, or of 32 narrow ones.
static unsigned pack_blocks(size_t n, size_t Kp) {
  size_t const b = Kp <= 256 ? n / 32 : n / 8;
  return static_cast<unsigned>(b < kCePackBlocks ? b : kCePackBlocks);
}

template <int NP>
CePlan ce_plan(dlmi_ctx const *ctx, size_t B, size_t K, size_t V, bool back) {
  CePlan p = {};
  // The tile with the least estimated time of all products: rounds of tiles over the CUs, the depth of their K loops, what 16 k
  // of a tile cost (measured, in us of two planes, of one plane a share of it; 128 and 64 wide tiles run two to a CU, where a CU
  // has one alone it is done sooner; many 64 wide ones wait for the L2) and its prologue and epilogue.  dX is cut into slices of
  // the classes that fill the device.  dW's tile is its own: [5789 x 415] FP32 against 17032 classes, whose dW has 68 tiles of
  // 256, went from 1790 to 1470 us.
  double const cu = ctx->num_cu;
  auto const product = [&](int t, double tiles, size_t k) {
    double const each = t == 256 ? 1.25 : t == 128 ? 0.35 : tiles <= 3 * cu ? 0.1 : 0.16, alone = t == 256 ? 1.25 : t == 128 ? 0.27 : 0.085;
    double const ends = t == 256 ? 12.0 : t == 128 ? 3.0 : 1.5;
    double const rounds = tiles / cu < 4.0 ? std::ceil(tiles / cu) : tiles / cu, depth = static_cast<double>(dlmi_ceil_div(k, 64) * 4);
    return rounds * ((tiles <= cu ? alone : each) * depth * (NP == 2 ? 1.0 : t == 256 ? 0.33 : 0.4) + ends);
  };
  auto const tiles_of = [](int t, size_t x, size_t y) { return static_cast<double>(dlmi_ceil_div(x, t)) * static_cast<double>(dlmi_ceil_div(y, t)); };
  double least = 0.0;
  for (int t : {256, 128, 64}) {
    double time = product(t, tiles_of(t, B, V), K);
    if (back) {
      double const n = tiles_of(t, B, K), full = std::max(n, cu * (t == 256 ? 1 : 2));
      time += product(t, full, static_cast<size_t>(static_cast<double>(V) * n / full));
    }
    if (t == 256 || time < least) {
      least = time;
      p.T = t;
    }
  }
  size_t const T = p.T;
  auto const up = [](size_t x, size_t m) { return dlmi_ceil_div(x, m) * m; };
  p.Bp = up(B, T);
  p.Kp = back ? up(K, T) : up(K, 64);
  // a piece: about four rounds of 256 wide tiles, eight of smaller ones, at most 1 GiB of packed operands
  size_t const nj = p.Bp / T;
  size_t tiles = dlmi_ceil_div(static_cast<size_t>(ctx->num_cu) * (T == 256 ? 4 : 8), nj);
  size_t const row_bytes = 2 * NP * (back ? 2 * (p.Kp + p.Bp) : p.Kp);
  size_t const fit = (size_t(1) << 30) / (row_bytes * T);
  if (tiles > fit) tiles = fit > 0 ? fit : 1;
  size_t const all = dlmi_ceil_div(V, T);
  p.pieces = dlmi_ceil_div(all, tiles);
  p.Vc = dlmi_ceil_div(all, p.pieces) * T;
  p.pieces = dlmi_ceil_div(V, p.Vc);
  for (int t : {256, 128, 64}) {
    if (t > p.T) continue;
    double const time = product(t, tiles_of(t, p.Vc, K), B);
    if (t == p.T || time < least) {
      least = time;
      p.Tw = t;
    }
  }
  size_t at = 0;
  auto const take = [&](size_t bytes) {
    size_t const o = at;
    at += up(bytes, 1024);
    return o;
  };
  p.xp = take(packed_bytes(p.Bp, p.Kp, NP));
  p.wp = take(packed_bytes(p.Vc, p.Kp, NP));
  p.pack_x = pack_blocks(p.Bp, p.Kp);
  p.pack_w = pack_blocks(p.Vc, p.Kp);
  p.unscale_x = take(p.Bp * sizeof(float));
  p.unscale_xw = take(p.Bp * sizeof(float));
  p.unscale_w = take(p.Vc * sizeof(float));
  p.parts_x = take(2 * p.pack_x * sizeof(float));
  p.most_x = take(2 * sizeof(float));
  p.most_w = take(2 * p.pieces * sizeof(float));
  if (!back) {
    p.part = take(dlmi_ceil_div(V, T) * 2 * p.Bp * sizeof(float2));
    p.target = take(B * sizeof(float));
  } else {
    p.xt = take(packed_bytes(p.Kp, p.Bp, NP));
    p.wt = take(packed_bytes(p.Kp, p.Vc, NP));
    p.dlb = take(packed_bytes(p.Bp, p.Vc, NP));  // (dL in fp32 takes the place of both, or of the first where NP is 2)
    p.dlv = take(packed_bytes(p.Vc, p.Bp, NP));
    size_t const dxt = p.Bp / T * (p.Kp / T), stages = dlmi_ceil_div(p.Vc, T == 64 ? 64 / NP : 32 / NP);
    size_t s = static_cast<size_t>(ctx->num_cu) * (T >= 256 ? 1 : 2) / dxt;
    if (s < 1) s = 1;
    if (s > 16) s = 16;
    if (s > stages / 16) s = stages / 16 > 0 ? stages / 16 : 1;
    p.per_slice = static_cast<unsigned>(dlmi_ceil_div(stages, s));
    p.slices = static_cast<unsigned>(dlmi_ceil_div(stages, p.per_slice));
    p.dxacc = take(p.slices * B * K * sizeof(float));
    p.dbpart = take(p.Bp / T * 2 * p.Vc * sizeof(float));
  }
  p.bytes = at;
  return p;
}

template <class E, int NP>
struct CeRun {
  dlmi_ctx *ctx;
  CeArgs a;
  CePlan p;
  char *s;

  // stages of the K loop over k values (padded rows of zeros follow them to a whole stage)
  static unsigned ce_stages(int T, size_t k) { return static_cast<unsigned>(dlmi_ceil_div(k, (T == 64 ? 64 : 32) / NP)); }
  float *floats(size_t at) const { return reinterpret_cast<float *>(s + at); }

  template <int KEEP, bool LABELS, bool ALONE>
  int pack(E const *src, size_t rows, size_t padded, unsigned blocks, size_t unscale, size_t piece, bool back, char *as, char *across) const {
    CeMost most = {};
    if (back) most = {floats(p.most_w), floats(p.most_x), floats(p.parts_x), p.pack_x, static_cast<unsigned>(piece), static_cast<unsigned>(p.pieces)};
    hipLaunchKernelGGL((k_ce_pack<E, NP, KEEP, LABELS, ALONE>), dim3(blocks), dim3(kCeBlock), 0, ctx->stream, a, src, rows, padded, a.K,
                       static_cast<unsigned>(p.Kp / 16), static_cast<unsigned>(padded / 16), floats(unscale), floats(p.unscale_xw),
                       most, as, across);
    DLMI_LAUNCH_CHECK(ctx, "k_ce_pack");
    return DLMI_OK;
  }
  int pack_rows(bool back) const {
    E const *const x = static_cast<E const *>(a.X);
    char *const across = back && a.dW != nullptr ? s + p.xt : nullptr;
    if (p.Kp <= 256) return pack<4, true, true>(x, a.B, p.Bp, p.pack_x, p.unscale_x, 0, back, s + p.xp, across);
    if (p.Kp <= 1024) return pack<4, true, false>(x, a.B, p.Bp, p.pack_x, p.unscale_x, 0, back, s + p.xp, across);
    return pack<8, true, false>(x, a.B, p.Bp, p.pack_x, p.unscale_x, 0, back, s + p.xp, across);
  }
  unsigned pack_w(size_t vp) const { return pack_blocks(vp, p.Kp) < p.pack_w ? pack_blocks(vp, p.Kp) : p.pack_w; }
  int pack_classes(size_t v0, size_t vn, size_t vp, bool back) const {
    E const *const w = static_cast<E const *>(a.W) + v0 * a.K;
    char *const across = back && a.dX != nullptr ? s + p.wt : nullptr;
    if (p.Kp <= 256) return pack<4, false, true>(w, vn, vp, pack_w(vp), p.unscale_w, v0 / p.Vc, back, s + p.wp, across);
    if (p.Kp <= 1024) return pack<4, false, false>(w, vn, vp, pack_w(vp), p.unscale_w, v0 / p.Vc, back, s + p.wp, across);
    return pack<8, false, false>(w, vn, vp, pack_w(vp), p.unscale_w, v0 / p.Vc, back, s + p.wp, across);
  }
  CeLogits logits(size_t v0, size_t vn, size_t vp) const {
    CeLogits g = {};
    g.P = s + p.wp;
    g.Q = s + p.xp;
    g.unscale_w = floats(p.unscale_w);
    g.unscale_x = floats(p.unscale_x);
    g.unscale_xw = floats(p.unscale_xw);
    g.most_x = floats(p.most_x);
    g.finest_x = g.most_x + 1;
    g.most_w = floats(p.most_w) + v0 / p.Vc;
    g.finest_w = g.most_w + p.pieces;
    g.dl = floats(p.dlb);
    g.dl_stride = vp;
    g.ni = static_cast<unsigned>(vp / p.T);
    g.nj = static_cast<unsigned>(p.Bp / p.T);
    g.kblocks = static_cast<unsigned>(p.Kp / 16);
    g.stages = ce_stages(p.T, a.K);
    g.v0 = v0;
    g.vn = vn;
    return g;
  }

  template <int T>
  int forward() const {
    int rc = pack_rows(false);
    for (size_t v0 = 0; rc == DLMI_OK && v0 < a.V; v0 += p.Vc) {
      size_t const vn = a.V - v0 < p.Vc ? a.V - v0 : p.Vc, vp = dlmi_ceil_div(vn, T) * T;
      rc = pack_classes(v0, vn, vp, false);
      if (rc != DLMI_OK) return rc;
      CeLogits const g = logits(v0, vn, vp);
      hipLaunchKernelGGL((k_ce_stats<T, NP>), dim3(g.ni * g.nj), dim3(256), 0, ctx->stream, a, g, reinterpret_cast<float2 *>(s + p.part), p.Bp,
                         v0 / T * 2, floats(p.target));
      DLMI_LAUNCH_CHECK(ctx, "k_ce_stats");
    }
    if (rc != DLMI_OK) return rc;
    hipLaunchKernelGGL(k_ce_join<16>, dim3(static_cast<unsigned>(dlmi_ceil_div(a.B, 16))), dim3(1024), 0, ctx->stream, a,
                       reinterpret_cast<float2 *>(s + p.part), p.Bp, dlmi_ceil_div(a.V, static_cast<size_t>(T)) * 2, floats(p.target));
    DLMI_LAUNCH_CHECK(ctx, "k_ce_join");
    return DLMI_OK;
  }

  // dW of a piece (tiles that are padding alone have no workgroup)
  template <int T>
  int weights(CeLogits const &g, size_t v0, size_t vn, unsigned kb) const {
    unsigned const ni = static_cast<unsigned>(dlmi_ceil_div(vn, T)), nk = static_cast<unsigned>(dlmi_ceil_div(a.K, T));
    hipLaunchKernelGGL((k_ce_dw<T, NP, E>), dim3(ni * nk), dim3(256), 0, ctx->stream, a, g, s + p.dlv, s + p.xt, ni, nk, kb, ce_stages(T, a.B),
                       a.scale, static_cast<E *>(a.dW) + v0 * a.K, vn, a.K, a.accumulate);
    DLMI_LAUNCH_CHECK(ctx, "k_ce_dw");
    return DLMI_OK;
  }

  template <int T>
  int backward() const {
    int rc = pack_rows(true);
    unsigned const nb = static_cast<unsigned>(p.Bp / T), nk = static_cast<unsigned>(p.Kp / T), kb = static_cast<unsigned>(p.Bp / 16);
    for (size_t v0 = 0; rc == DLMI_OK && v0 < a.V; v0 += p.Vc) {
      size_t const vn = a.V - v0 < p.Vc ? a.V - v0 : p.Vc, vp = dlmi_ceil_div(vn, T) * T;
      rc = pack_classes(v0, vn, vp, true);
      if (rc != DLMI_OK) return rc;
      CeLogits const g = logits(v0, vn, vp);
      unsigned const kv = static_cast<unsigned>(vp / 16);
      if (a.db != nullptr)
        hipLaunchKernelGGL((k_ce_grad<T, NP, true>), dim3(g.ni * g.nj), dim3(256), 0, ctx->stream, a, g, s + p.dlb, s + p.dlv, kv, kb,
                           floats(p.dbpart), p.Vc);
      else
        hipLaunchKernelGGL((k_ce_grad<T, NP, false>), dim3(g.ni * g.nj), dim3(256), 0, ctx->stream, a, g, s + p.dlb, s + p.dlv, kv, kb,
                           nullptr, p.Vc);
      DLMI_LAUNCH_CHECK(ctx, "k_ce_grad");
      if (a.db != nullptr) {
        hipLaunchKernelGGL(k_ce_db, dim3(static_cast<unsigned>(dlmi_ceil_div(vn, kCeBlock))), dim3(kCeBlock), 0, ctx->stream, floats(p.dbpart),
                           p.Vc, nb * 2, vn, a.db + v0, a.scale, a.accumulate);
        DLMI_LAUNCH_CHECK(ctx, "k_ce_db");
      }
      if (a.dX != nullptr) {
        hipLaunchKernelGGL((k_ce_dx<T, NP, E>), dim3(nb * nk * p.slices), dim3(256), 0, ctx->stream, g, static_cast<E const *>(a.W) + v0 * a.K,
                           s + p.dlb, s + p.wt, nb, nk, kv, ce_stages(T, vp), p.per_slice, floats(p.dxacc), a.B, a.K, v0 == 0 ? 1 : 0);
        DLMI_LAUNCH_CHECK(ctx, "k_ce_dx");
      }
      if (a.dW != nullptr) {
        if (p.Tw == T)
          rc = weights<T>(g, v0, vn, kb);
        else if (p.Tw == 128)
          rc = weights<128>(g, v0, vn, kb);
        else
          rc = weights<64>(g, v0, vn, kb);
      }
    }
    if (rc != DLMI_OK || a.dX == nullptr) return rc;
    dim3 const grid(static_cast<unsigned>(a.B), static_cast<unsigned>(dlmi_ceil_div(a.K, kCeBlock * 4)));
    hipLaunchKernelGGL(k_ce_dx_finish<E>, grid, dim3(kCeBlock), 0, ctx->stream, a, floats(p.dxacc), p.slices, static_cast<E *>(a.dX));
    DLMI_LAUNCH_CHECK(ctx, "k_ce_dx_finish");
    return DLMI_OK;
  }
};

template <class E>
constexpr int kCePlanes = sizeof(E) == 4 ? 2 : 1;

template <class E>
static int ce_run(dlmi_ctx *ctx, CeArgs const &a, bool back) {
  constexpr int NP = kCePlanes<E>;
  CeRun<E, NP> r{ctx, a, ce_plan<NP>(ctx, a.B, a.K, a.V, back), nullptr};
  int const rc = dlmi_scratch_reserve(ctx, r.p.bytes);
  if (rc != DLMI_OK) return rc;
  r.s = dlmi_scratch_data(ctx);
  switch (r.p.T) {
    case 256: return back ? r.template backward<256>() : r.template forward<256>();
    case 128: return back ? r.template backward<128>() : r.template forward<128>();
    default: return back ? r.template backward<64>() : r.template forward<64>();
  }
}

template <class E, int RB, int VB, int NB, int NW>
static int ce_direct(dlmi_ctx *ctx, CeArgs const &a, int per_cu) {
  // as many workgroups as run at once
  size_t const most = static_cast<size_t>(ctx->num_cu) * per_cu;
  size_t const all = dlmi_ceil_div(a.V, RB * VB), blocks = all < most ? all : most;
  size_t const bytes = blocks * a.B * sizeof(float2);
  int const rc = dlmi_scratch_reserve(ctx, bytes + a.B * sizeof(float));
  if (rc != DLMI_OK) return rc;
  char *const s = dlmi_scratch_data(ctx);
  hipLaunchKernelGGL((k_ce_direct<E, RB, VB, NB, NW>), dim3(static_cast<unsigned>(blocks)), dim3(NW * 64), 0, ctx->stream, a,
                     reinterpret_cast<float2 *>(s), reinterpret_cast<float *>(s + bytes), ctx->pair_ticket);
  DLMI_LAUNCH_CHECK(ctx, "k_ce_direct");
  return DLMI_OK;
}

template <class E>
int ce_forward(dlmi_ctx *ctx, CeArgs const &a) {
  // 64 classes a workgroup where that still gives every CU two
  bool const wide = dlmi_ceil_div(a.V, 64) >= static_cast<size_t>(ctx->num_cu) * 2;
  if (a.B <= 16) return wide ? ce_direct<E, 16, 4, 1, 8>(ctx, a, 1) : ce_direct<E, 16, 2, 1, 8>(ctx, a, 2);
  if (a.B <= 32) return wide ? ce_direct<E, 32, 2, 1, 8>(ctx, a, 1) : ce_direct<E, 32, 1, 1, 8>(ctx, a, 2);
  if (a.B <= 64) return wide ? ce_direct<E, 32, 2, 2, 4>(ctx, a, 2) : ce_direct<E, 32, 1, 2, 8>(ctx, a, 1);
  return ce_run<E>(ctx, a, false);
}
template <class E>
int ce_backward(dlmi_ctx *ctx, CeArgs const &a) {
  return ce_run<E>(ctx, a, true);
}

#endif  // DLMI_CE_IMPLEMENTATION

}  // namespace dlmi
