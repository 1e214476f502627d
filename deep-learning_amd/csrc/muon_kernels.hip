// Newton-Schulz orthogonalization of a matrix and the Muon optimizer step built on it, for gfx950.
//
//   m <- momentum m + g;  u = nesterov ? g + momentum m : m
//   X <- u / (|u|_F + eps), on its short side (transposed when rows > cols)
//   `steps` times:  A = X X^T;  X <- a X + (b A + c A A) X
//   p <- p - lr X - wd p
//
// Each step maps the singular values of X by a s + b s^3 + c s^5 and leaves its singular vectors: all of them end near 1.
// Bound by the 16-bit matrix pipe: per step s^2 l (X X^T, half of it: A is symmetric) + s^3 (A A, half) + 2 s^2 l
// operations, s the short and l the long side, times three for the two planes of half_gemm.hpp.
//
// Precision.  The polynomial multiplies what lies in weak directions by up to a^steps (485 for 5 steps of 3.4445), the
// rounding of the operands among it.  With one f16 plane a random matrix ends 1.3e-3 off and a matrix of rank 32 plus 1 %
// noise 2.7e-2; with two planes (22 bits) 1.8e-6 and 1.2e-5, as far as a computation in fp32 (1.1e-5 and 1.9e-5).  So X,
// A and a I + b A + c A A keep two planes in every step.  (One plane in the last step of a bf16 result adds 4.5e-4 to 1.0e-3 to
// the 1.7e-3 of rounding it, in the norm, but rounds one element in five to another value, small ones up to 60 half steps
// away; it saved a tenth of a 4096 x 4096 call.)  16 x 2048 x 2048 FP32: 8.1 - 8.3 ms a step; 4096 x 4096 BF16: 3.8 ms; 1531 x
// 517 BF16: 150 us; 128 x 256: 77 - 87 us, 17 launches of 3.4 to 5.4.  Singular values stay below about 1.3 and the polynomial in
// A between -3 and 4, so all three matrices are held times 2^12: far from the ends of f16's range.
//
// X is kept both ways round (rows i, k = j for X X^T; rows j, k = i for the product by X), each written by the product
// that makes it: a block of C in registers is a fragment of the transposed matrix as it stands, and two matrix
// instructions by the identity turn it.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "half_gemm.hpp"

namespace dlmi {

constexpr int kMuonMax = 32;         // matrices per launch
constexpr int kMuonBlock = 256;
constexpr float kMuonScale = 4096.0f;

struct MuonBatch {
  void *p[kMuonMax];        // parameters (step) or output (orthogonalize)
  void *g[kMuonMax];        // gradient or input
  float *m[kMuonMax];
  float lr[kMuonMax];
};

__device__ __forceinline__ double muon_block_sum(double s, double *lds) {
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  s = (lds[0] + lds[1]) + (lds[2] + lds[3]);
  __syncthreads();
  return s;
}

// Bound by memory: 151 us for 16 matrices of 2048 x 2048 = 5.3 TB/s.  The momentum, and partial[matrix][block] = sum of u^2 (double: the norm of a tiny gradient does not underflow).  Four
// elements of a thread at a time: their loads are on their way together.
template <class T, bool STEP>
__global__ __launch_bounds__(kMuonBlock) void k_muon_moment(MuonBatch b, size_t n, float momentum, int nesterov, double *partial) {
  __shared__ double lds[kMuonBlock / 64];
  struct __attribute__((packed, aligned(sizeof(T)))) V {
    T v[4];
  };
  struct __attribute__((packed, aligned(4))) F {
    float v[4];
  };
  T const *const g = static_cast<T const *>(b.g[blockIdx.y]);
  float *const m = b.m[blockIdx.y];
  auto const one = [&](float x, float &mv) {
    if constexpr (STEP) {
      mv = momentum * mv + x;
      x = nesterov ? x + momentum * mv : mv;
    }
    return static_cast<double>(x) * x;
  };
  size_t const quads = n / 4, stride = static_cast<size_t>(gridDim.x) * kMuonBlock;
  size_t const at = static_cast<size_t>(blockIdx.x) * kMuonBlock + threadIdx.x;
  double s = 0.0;
#pragma unroll 2
  for (size_t i = at; i < quads; i += stride) {
    V const x = *reinterpret_cast<V const *>(g + i * 4);
    F w = {};
    if constexpr (STEP) w = *reinterpret_cast<F const *>(m + i * 4);
    double q = 0.0;
#pragma unroll
    for (int t = 0; t < 4; ++t) q += one(static_cast<float>(x.v[t]), w.v[t]);
    if constexpr (STEP) *reinterpret_cast<F *>(m + i * 4) = w;
    s += q;
  }
  if (at < n - quads * 4) {
    float w = 0.0f;
    if constexpr (STEP) w = m[quads * 4 + at];
    s += one(static_cast<float>(g[quads * 4 + at]), w);
    if constexpr (STEP) m[quads * 4 + at] = w;
  }
  s = muon_block_sum(s, lds);
  if (threadIdx.x == 0) partial[static_cast<size_t>(blockIdx.y) * gridDim.x + blockIdx.x] = s;
}

// One 64 x 64 tile of u / (|u| + eps), packed as it stands (row r, k = c: `rc`) and transposed (row c, k = r: `cr`);
// padding is zero.  A step's gradient is cleared on the way.  Bound by memory: 250 us for 16 matrices of 2048 x 2048 = 5.4 TB/s.
template <class T, bool STEP>
__global__ __launch_bounds__(kMuonBlock) void k_muon_pack(MuonBatch b, unsigned R, unsigned C, unsigned Rp, unsigned Cp, float momentum,
                                                          int nesterov, float eps, double const *partial, unsigned nparts, char *rc,
                                                          char *cr, size_t stride) {
  __shared__ double sums[kMuonBlock / 64];
  __shared__ float tile[64][65];
  unsigned const mat = blockIdx.z;
  double s = 0.0;
  for (unsigned i = threadIdx.x; i < nparts; i += kMuonBlock) s += partial[static_cast<size_t>(mat) * nparts + i];
  s = muon_block_sum(s, sums);
  double const inv = static_cast<double>(kMuonScale) / (sqrt(s) + static_cast<double>(eps));  // double: of a tiny gradient it passes fp32's range
  T *const g = static_cast<T *>(b.g[mat]);
  float const *const m = b.m[mat];
  unsigned const r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;
  // every load is made, of the last row and column at most: loads behind conditions of their own would each be waited for
  unsigned const tc = threadIdx.x & 63, c = c0 + tc, cl = c < C ? c : C - 1;
  float gv[16], mv[16];
#pragma unroll
  for (int q = 0; q < 16; ++q) {
    unsigned const r = r0 + q * 4 + (threadIdx.x >> 6);
    size_t const at = static_cast<size_t>(r < R ? r : R - 1) * C + cl;
    gv[q] = static_cast<float>(g[at]);
    mv[q] = STEP ? m[at] : 0.0f;
  }
#pragma unroll
  for (int q = 0; q < 16; ++q) {
    unsigned const tr = q * 4 + (threadIdx.x >> 6), r = r0 + tr;
    bool const in = r < R && c < C;
    float u = gv[q];
    if constexpr (STEP) {
      u = nesterov ? u + momentum * mv[q] : mv[q];
      if (in) g[static_cast<size_t>(r) * C + c] = static_cast<T>(0.0f);
    }
    tile[tr][tc] = in ? static_cast<float>(u * inv) : 0.0f;
  }
  __syncthreads();
  int const lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  char *const drc = rc + mat * stride, *const dcr = cr + mat * stride;
  unsigned const kbs = Cp / 16, kbr = Rp / 16;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    int const f = q * 4 + wave;       // 16 fragments: 8 as it stands, 8 transposed
    bool const flip = f >= 8;
    int const rb = (f >> 2) & 1, kb = f & 3;
    half8 hi, lo;
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      int const row = rb * 32 + (lane & 31), k = kb * 16 + (lane >> 5) * 8 + t;
      float x = flip ? tile[k][row] : tile[row][k];
      asm("" : "+v"(x));  // (one value for both planes)
      _Float16 const h = static_cast<_Float16>(x);
      hi[t] = h;
      lo[t] = static_cast<_Float16>(x - static_cast<float>(h));
    }
    size_t const frag = flip ? static_cast<size_t>(c0 / 32 + rb) * kbr + r0 / 16 + kb : static_cast<size_t>(r0 / 32 + rb) * kbs + c0 / 16 + kb;
    char *const dst = (flip ? dcr : drc) + frag * 2 * kFragBytes + lane * 16;
    *reinterpret_cast<half8 *>(dst) = hi;
    *reinterpret_cast<half8 *>(dst + kFragBytes) = lo;
  }
}

// A tile of a symmetric product C = P P^T (P: [mp, k] packed), only the tiles on and below the diagonal; written packed
// with its mirror image.  16 matrices of 2048 x 2048: 340 us and 70 for the shared last tiles = 1130 TFLOP/s of 16-bit
// products.  POLY: C = a I + b P + c P P^T (P symmetric itself).  Products of two values held times 2^12.
struct MuonSymmetric {
  char const *P;
  char *C;
  size_t stride_p, stride_c;
  unsigned tiles, kblocks, kblocks_c;  // of a side; k blocks of P and of C
  float ca, cb, cc;
};

__device__ __forceinline__ void muon_triangle(unsigned t, unsigned &ti, unsigned &tj) {
  ti = static_cast<unsigned>((sqrtf(8.0f * static_cast<float>(t) + 1.0f) - 1.0f) * 0.5f);
  while (ti * (ti + 1) / 2 > t) --ti;
  while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
  tj = t - ti * (ti + 1) / 2;
}

template <bool POLY>
__device__ __forceinline__ void muon_symmetric_block(MuonSymmetric const &a, unsigned mat, unsigned ib, unsigned jb, bool mirror, f32x16 v,
                                                     half8 id0, half8 id1, int lane) {
  char const *const p = a.P + mat * a.stride_p;
  char *const c = a.C + mat * a.stride_c;
  size_t const rs = static_cast<size_t>(a.kblocks) * 2 * kFragBytes, rc = static_cast<size_t>(a.kblocks_c) * 2 * kFragBytes;
  v *= a.cc / kMuonScale;
  if constexpr (POLY) {
    v += a.cb * half_load<2>(p + jb * rs + ib * 4 * kFragBytes, lane);
    if (ib == jb) {
#pragma unroll
      for (int r = 0; r < 16; ++r) v[r] += 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3) == (lane & 31) ? a.ca * kMuonScale : 0.0f;
    }
  }
  HalfBlock<2> const blk = half_split<2>(v);
  half_store<2>(c + jb * rc + ib * 4 * kFragBytes, blk, lane);
  if (mirror) half_store<2>(c + ib * rc + jb * 4 * kFragBytes, half_flip<2>(blk, id0, id1), lane);
}

struct MuonTile {
  unsigned mat, ti, tj;
};
__device__ __forceinline__ MuonTile muon_tile(MuonSymmetric const &a, unsigned tile) {
  unsigned const tri = a.tiles * (a.tiles + 1) / 2;
  MuonTile t;
  t.mat = tile / tri;
  muon_triangle(tile - t.mat * tri, t.ti, t.tj);
  return t;
}

template <int T, bool POLY>
__global__ __launch_bounds__(256, T >= 256 ? 1 : 2) void k_muon_symmetric(MuonSymmetric a, unsigned stages) {
  using H = HalfTile<T, T, 2>;
  MuonTile const t = muon_tile(a, xcd_consecutive(blockIdx.x, gridDim.x));
  size_t const rs = static_cast<size_t>(a.kblocks) * 2 * kFragBytes;
  char const *const p = a.P + t.mat * a.stride_p;
  HalfAcc<H> acc;
  half_gemm<H>(acc, p + t.ti * (T / 32) * rs, p + t.tj * (T / 32) * rs, rs, rs, stages);
  int const lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  half8 const id0 = half_identity(0, lane), id1 = half_identity(1, lane);
#pragma unroll
  for (int m = 0; m < H::kMB; ++m)
#pragma unroll
    for (int n = 0; n < H::kNB; ++n)
      muon_symmetric_block<POLY>(a, t.mat, t.ti * (T / 32) + (wave >> 1) * H::kMB + m, t.tj * (T / 32) + (wave & 1) * H::kNB + n, t.ti != t.tj,
                                 acc.v[m][n], id0, id1, lane);
}

template <int T>
__global__ __launch_bounds__(256, 1) void k_muon_symmetric_parts(MuonSymmetric a, HalfShares shares) {
  size_t const rs = static_cast<size_t>(a.kblocks) * 2 * kFragBytes;
  half_gemm_parts<HalfTile<T, T, 2>>(shares, rs, rs, [&](unsigned tile, char const *&p, char const *&q) {
    MuonTile const t = muon_tile(a, tile);
    p = a.P + t.mat * a.stride_p + t.ti * (T / 32) * rs;
    q = a.P + t.mat * a.stride_p + t.tj * (T / 32) * rs;
  });
}

// The blocks of the shared tiles, a wavefront each.
template <int T, bool POLY>
__global__ __launch_bounds__(256) void k_muon_symmetric_join(MuonSymmetric a, HalfShares shares) {
  using H = HalfTile<T, T, 2>;
  constexpr unsigned kBlocks = (T / 32) * (T / 32), kWave = H::kMB * H::kNB;
  int const lane = threadIdx.x & 63;
  unsigned const id = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), shared = id / kBlocks, block = id % kBlocks;
  f32x16 const v = half_part_sum<H>(shares, shared, block, T * T);
  MuonTile const t = muon_tile(a, shares.whole + shared);
  unsigned const wave = block / kWave, m = block % kWave / H::kNB, n = block % H::kNB;
  muon_symmetric_block<POLY>(a, t.mat, t.ti * (T / 32) + (wave >> 1) * H::kMB + m, t.tj * (T / 32) + (wave & 1) * H::kNB + n, t.ti != t.tj, v,
                             half_identity(0, lane), half_identity(1, lane), lane);
}

enum { kMuonMore = 0, kMuonOut = 1, kMuonStep = 2 };

struct MuonOut {
  unsigned rows, cols;   // of the caller's matrix
  int flipped;           // X is the transposed matrix
  float wd;
};

template <int MODE>
__device__ __forceinline__ float muon_new(float w, float x, float lr, float wd) {
  return MODE == kMuonStep ? w - (lr * x + wd * w) : x;
}

// A tile of X' = Bm X, Bm = a I + b A + c A A (a X inside the product: read beside it in the epilogue it is 4 bytes more per
// element, while the matrix pipe waits); XT = X^T packed (row j, k = i).  MORE: written packed both ways; OUT, STEP: the last of the
// iteration, written to the caller's matrix.  16 matrices of 2048 x 2048: 681 us = 1210 TFLOP/s of 16-bit products.
struct MuonUpdate {
  char const *Bm, *XT;
  char *XTn, *XP;
  size_t stride_b, stride_x;
  unsigned mt, nt, kbm, kbn;  // tiles and k blocks of the short and of the long side
  MuonOut o;
};

template <int MODE, class O>
__device__ __forceinline__ void muon_update_block(MuonUpdate const &a, MuonBatch const &b, unsigned mat, unsigned ib, unsigned jb, f32x16 v,
                                                  half8 id0, half8 id1, int lane) {
  size_t const rs = static_cast<size_t>(a.kbm) * 2 * kFragBytes, rn = static_cast<size_t>(a.kbn) * 2 * kFragBytes;
  v *= 1.0f / kMuonScale;
  if constexpr (MODE == kMuonMore) {
    HalfBlock<2> const blk = half_split<2>(v);
    half_store<2>(a.XTn + mat * a.stride_x + jb * rs + ib * 4 * kFragBytes, blk, lane);
    half_store<2>(a.XP + mat * a.stride_x + ib * rn + jb * 4 * kFragBytes, half_flip<2>(blk, id0, id1), lane);
  } else {
    MuonOut const &o = a.o;
    v *= 1.0f / kMuonScale;
    O *const p = static_cast<O *>(b.p[mat]);
    size_t const j = jb * 32 + (lane & 31), i0 = ib * 32 + 4 * (lane >> 5);
    size_t const si = o.flipped ? 1 : o.cols, sj = o.flipped ? o.cols : 1;
    unsigned const rows = o.flipped ? o.cols : o.rows, cols = o.flipped ? o.rows : o.cols;  // of X
    float const lr = MODE == kMuonStep ? b.lr[mat] : 0.0f;
    // (a block inside the matrix has no conditions between its loads, which would each be waited for)
    if (ib * 32 + 32 <= rows && jb * 32 + 32 <= cols) {
      O *const q = p + i0 * si + j * sj;
      f32x16 w = {};
      if constexpr (MODE == kMuonStep) {
#pragma unroll
        for (int r = 0; r < 16; ++r) w[r] = static_cast<float>(q[(8 * (r >> 2) + (r & 3)) * si]);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) q[(8 * (r >> 2) + (r & 3)) * si] = static_cast<O>(muon_new<MODE>(w[r], v[r], lr, o.wd));
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        size_t const i = i0 + 8 * (r >> 2) + (r & 3);
        if (i < rows && j < cols) {
          O *const q = p + i * si + j * sj;
          *q = static_cast<O>(muon_new<MODE>(MODE == kMuonStep ? static_cast<float>(*q) : 0.0f, v[r], lr, o.wd));
        }
      }
    }
  }
}

__device__ __forceinline__ MuonTile muon_tile(MuonUpdate const &a, unsigned tile) {
  MuonTile t;
  t.mat = tile / (a.mt * a.nt);
  unsigned const r = tile - t.mat * (a.mt * a.nt);
  t.tj = r / a.mt;
  t.ti = r - t.tj * a.mt;
  return t;
}

template <int T, int MODE, class O>
__global__ __launch_bounds__(256, T >= 256 ? 1 : 2) void k_muon_update(MuonUpdate a, MuonBatch b, unsigned stages) {
  using H = HalfTile<T, T, 2>;
  MuonTile const t = muon_tile(a, xcd_consecutive(blockIdx.x, gridDim.x));
  size_t const rs = static_cast<size_t>(a.kbm) * 2 * kFragBytes;
  HalfAcc<H> acc;
  half_gemm<H>(acc, a.Bm + t.mat * a.stride_b + t.ti * (T / 32) * rs, a.XT + t.mat * a.stride_x + t.tj * (T / 32) * rs, rs, rs, stages);
  int const lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  half8 const id0 = half_identity(0, lane), id1 = half_identity(1, lane);
#pragma unroll
  for (int m = 0; m < H::kMB; ++m)
#pragma unroll
    for (int n = 0; n < H::kNB; ++n)
      muon_update_block<MODE, O>(a, b, t.mat, t.ti * (T / 32) + (wave >> 1) * H::kMB + m, t.tj * (T / 32) + (wave & 1) * H::kNB + n,
                                 acc.v[m][n], id0, id1, lane);
}

template <int T>
__global__ __launch_bounds__(256, 1) void k_muon_update_parts(MuonUpdate a, HalfShares shares) {
  size_t const rs = static_cast<size_t>(a.kbm) * 2 * kFragBytes;
  half_gemm_parts<HalfTile<T, T, 2>>(shares, rs, rs, [&](unsigned tile, char const *&p, char const *&q) {
    MuonTile const t = muon_tile(a, tile);
    p = a.Bm + t.mat * a.stride_b + t.ti * (T / 32) * rs;
    q = a.XT + t.mat * a.stride_x + t.tj * (T / 32) * rs;
  });
}

template <int T, int MODE, class O>
__global__ __launch_bounds__(256) void k_muon_update_join(MuonUpdate a, MuonBatch b, HalfShares shares) {
  using H = HalfTile<T, T, 2>;
  constexpr unsigned kBlocks = (T / 32) * (T / 32), kWave = H::kMB * H::kNB;
  int const lane = threadIdx.x & 63;
  unsigned const id = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), shared = id / kBlocks, block = id % kBlocks;
  f32x16 const v = half_part_sum<H>(shares, shared, block, T * T);
  MuonTile const t = muon_tile(a, shares.whole + shared);
  unsigned const wave = block / kWave, m = block % kWave / H::kNB, n = block % H::kNB;
  muon_update_block<MODE, O>(a, b, t.mat, t.ti * (T / 32) + (wave >> 1) * H::kMB + m, t.tj * (T / 32) + (wave & 1) * H::kNB + n, v,
                             half_identity(0, lane), half_identity(1, lane), lane);
}

// The iteration's bounds for singular values in [0, 1]: largest magnitude of X X^T and of a I + b A + c A A on the way.
static double muon_reach(float const *coefs, int steps) {
  double most = 1.0;
  for (int i = 0; i <= 2048; ++i) {
    double s = i / 2048.0;
    for (int k = 0; k < steps; ++k) {
      double const q = s * s, poly = coefs[0] + coefs[1] * q + coefs[2] * q * q;
      s *= poly;
      if (!(std::fabs(poly) <= 1e6) || !(std::fabs(s) <= 1e6)) return 1e6;
      if (std::fabs(poly) > most) most = std::fabs(poly);
      if (s * s > most) most = s * s;
    }
  }
  return most;
}

struct MuonPlan {
  int flipped;
  size_t mp, np, bytes_x, bytes_a, per_matrix;
  int tile;
  unsigned nparts;
  unsigned workgroups;         // that run at once
  size_t parts;                // bytes of the parts of shared tiles
  size_t bytes(size_t count) const { return per_matrix * count + parts; }
};

// Stages of a K loop that are worth sharing by the whole device.
static double muon_long_loop(int tile) { return tile == 128 ? 50.0 : 80.0; }

static MuonPlan muon_plan(dlmi_ctx const *ctx, size_t rows, size_t cols, size_t count) {
  MuonPlan pl;
  pl.flipped = rows > cols;
  size_t const s = pl.flipped ? cols : rows, l = pl.flipped ? rows : cols;
  pl.tile = 64;
  for (int T : {256, 128}) {
    size_t const tiles = dlmi_ceil_div(s, T) * dlmi_ceil_div(l, T) * count;
    if (tiles >= static_cast<size_t>(ctx->num_cu) * 3 / 4) {
      pl.tile = T;
      break;
    }
  }
  pl.mp = dlmi_ceil_div(s, pl.tile) * pl.tile;
  pl.np = dlmi_ceil_div(l, pl.tile) * pl.tile;
  pl.bytes_x = packed_bytes(pl.mp, pl.np, 2);
  pl.bytes_a = packed_bytes(pl.mp, pl.mp, 2);
  pl.nparts = static_cast<unsigned>(dlmi_ceil_div(rows * cols, kMuonBlock * 8));
  if (pl.nparts > 256) pl.nparts = 256;
  pl.per_matrix = 3 * pl.bytes_x + 2 * pl.bytes_a + dlmi_ceil_div(pl.nparts * sizeof(double), 1024) * 1024;
  // a workgroup per CU for tiles that are shared out, two parts each
  pl.workgroups = static_cast<unsigned>(ctx->num_cu);
  bool const may = pl.tile == 256 || static_cast<double>(pl.np / (pl.tile == 128 ? 16 : 32)) > muon_long_loop(pl.tile);
  pl.parts = may ? static_cast<size_t>(pl.workgroups) * 2 * pl.tile * pl.tile * sizeof(float) : 0;
  return pl;
}

// Whether sharing out the last tiles pays for the second launch and the parts' way through memory.  256 x 256 tiles: where
// their round is at most three quarters full.  Smaller ones: where they are too few for the device and their K loops long,
// which a CU walks at what it takes from the L2, about 0.27 us a stage of 128 x 128 and 0.17 of 64 x 64 (eleven matrices of
// 112 x 3141: 386 -> 282 us a step; 1531 x 517, whose loops have 48 stages, would go from 146 to 156: a launch and the parts
// cost as much as 13 us of a loop).
static HalfShares muon_shares(MuonPlan const &pl, unsigned tiles, unsigned stages, float *parts) {
  unsigned const over = tiles % pl.workgroups;
  bool share = over != 0 && over * 4 <= pl.workgroups * 3;
  if (pl.tile != 256) share = tiles < pl.workgroups && stages * (1.0 - static_cast<double>(tiles) / pl.workgroups) > muon_long_loop(pl.tile);
  return half_shares(tiles, stages, share ? pl.workgroups : tiles, parts);
}

template <int T, bool POLY>
static int muon_symmetric(dlmi_ctx *ctx, MuonSymmetric const &a, HalfShares const &shares) {
  if (shares.whole != 0) {
    hipLaunchKernelGGL((k_muon_symmetric<T, POLY>), dim3(shares.whole), dim3(256), 0, ctx->stream, a, shares.stages);
    DLMI_LAUNCH_CHECK(ctx, "k_muon_symmetric");
  }
  if (shares.total == 0) return DLMI_OK;
  hipLaunchKernelGGL((k_muon_symmetric_parts<T>), dim3(shares.grid), dim3(256), 0, ctx->stream, a, shares);
  DLMI_LAUNCH_CHECK(ctx, "k_muon_symmetric_parts");
  unsigned const blocks = (shares.tiles - shares.whole) * (T / 32) * (T / 32) / 4;
  hipLaunchKernelGGL((k_muon_symmetric_join<T, POLY>), dim3(blocks), dim3(256), 0, ctx->stream, a, shares);
  DLMI_LAUNCH_CHECK(ctx, "k_muon_symmetric_join");
  return DLMI_OK;
}

template <int T, int MODE, class O>
static int muon_update(dlmi_ctx *ctx, MuonUpdate const &a, MuonBatch const &b, HalfShares const &shares) {
  if (shares.whole != 0) {
    hipLaunchKernelGGL((k_muon_update<T, MODE, O>), dim3(shares.whole), dim3(256), 0, ctx->stream, a, b, shares.stages);
    DLMI_LAUNCH_CHECK(ctx, "k_muon_update");
  }
  if (shares.total == 0) return DLMI_OK;
  hipLaunchKernelGGL((k_muon_update_parts<T>), dim3(shares.grid), dim3(256), 0, ctx->stream, a, shares);
  DLMI_LAUNCH_CHECK(ctx, "k_muon_update_parts");
  unsigned const blocks = (shares.tiles - shares.whole) * (T / 32) * (T / 32) / 4;
  hipLaunchKernelGGL((k_muon_update_join<T, MODE, O>), dim3(blocks), dim3(256), 0, ctx->stream, a, b, shares);
  DLMI_LAUNCH_CHECK(ctx, "k_muon_update_join");
  return DLMI_OK;
}

// A step of the iteration.
template <int T, int MODE, class O>
static int muon_one(dlmi_ctx *ctx, MuonPlan const &pl, MuonBatch const &b, MuonSymmetric const &g, MuonSymmetric const &q, MuonUpdate const &u,
                    unsigned count, float *parts) {
  constexpr unsigned KS = HalfTile<T, T, 2>::KS;
  unsigned const tri = u.mt * (u.mt + 1) / 2 * count;
  int rc = muon_symmetric<T, false>(ctx, g, muon_shares(pl, tri, u.kbn / KS, parts));
  if (rc == DLMI_OK) rc = muon_symmetric<T, true>(ctx, q, muon_shares(pl, tri, u.kbm / KS, parts));
  if (rc == DLMI_OK) rc = muon_update<T, MODE, O>(ctx, u, b, muon_shares(pl, u.mt * u.nt * count, u.kbm / KS, parts));
  return rc;
}

template <int T, class O, bool STEP>
static int muon_iterate(dlmi_ctx *ctx, MuonBatch const &b, MuonPlan const &pl, unsigned count, float const *coefs, int steps,
                        MuonOut const &o, char *XP, char *XT, char *XTn, char *A, char *Bm, float *parts) {
  unsigned const mt = static_cast<unsigned>(pl.mp / T), nt = static_cast<unsigned>(pl.np / T);
  unsigned const kbm = static_cast<unsigned>(pl.mp / 16), kbn = static_cast<unsigned>(pl.np / 16);
  MuonSymmetric const g{XP, A, pl.bytes_x, pl.bytes_a, mt, kbn, kbm, 0.0f, 0.0f, 1.0f};
  MuonSymmetric const q{A, Bm, pl.bytes_a, pl.bytes_a, mt, kbm, kbm, coefs[0], coefs[1], coefs[2]};
  MuonUpdate u{Bm, XT, XTn, XP, pl.bytes_a, pl.bytes_x, mt, nt, kbm, kbn, o};
  for (int s = 0; s + 1 < steps; ++s) {
    int const rc = muon_one<T, kMuonMore, O>(ctx, pl, b, g, q, u, count, parts);
    if (rc != DLMI_OK) return rc;
    char *const x = const_cast<char *>(u.XT);
    u.XT = u.XTn;
    u.XTn = x;
  }
  return muon_one<T, STEP ? kMuonStep : kMuonOut, O>(ctx, pl, b, g, q, u, count, parts);
}

// `count` matrices of one shape, at most kMuonMax of them; the scratch has been reserved.
template <class T, bool STEP>
static int muon_batch(dlmi_ctx *ctx, MuonBatch const &b, size_t rows, size_t cols, unsigned count, MuonPlan const &pl, float momentum,
                      int nesterov, float wd, int steps, float const *coefs, float eps) {
  char *const XP = dlmi_scratch_data(ctx), *const XT = XP + count * pl.bytes_x, *const XTn = XT + count * pl.bytes_x;
  char *const A = XTn + count * pl.bytes_x, *const Bm = A + count * pl.bytes_a;
  float *const parts = reinterpret_cast<float *>(Bm + count * pl.bytes_a);
  double *const partial = reinterpret_cast<double *>(reinterpret_cast<char *>(parts) + pl.parts);
  size_t const n = rows * cols;
  hipLaunchKernelGGL((k_muon_moment<T, STEP>), dim3(pl.nparts, count), dim3(kMuonBlock), 0, ctx->stream, b, n, momentum, nesterov, partial);
  DLMI_LAUNCH_CHECK(ctx, "k_muon_moment");
  size_t const Rp = pl.flipped ? pl.np : pl.mp, Cp = pl.flipped ? pl.mp : pl.np;
  hipLaunchKernelGGL((k_muon_pack<T, STEP>), dim3(static_cast<unsigned>(Cp / 64), static_cast<unsigned>(Rp / 64), count), dim3(kMuonBlock), 0,
                     ctx->stream, b, static_cast<unsigned>(rows), static_cast<unsigned>(cols), static_cast<unsigned>(Rp),
                     static_cast<unsigned>(Cp), momentum, nesterov, eps, partial, pl.nparts, pl.flipped ? XT : XP, pl.flipped ? XP : XT,
                     pl.bytes_x);
  DLMI_LAUNCH_CHECK(ctx, "k_muon_pack");
  MuonOut const o{static_cast<unsigned>(rows), static_cast<unsigned>(cols), pl.flipped, wd};
  if (pl.tile == 256) return muon_iterate<256, T, STEP>(ctx, b, pl, count, coefs, steps, o, XP, XT, XTn, A, Bm, parts);
  if (pl.tile == 128) return muon_iterate<128, T, STEP>(ctx, b, pl, count, coefs, steps, o, XP, XT, XTn, A, Bm, parts);
  return muon_iterate<64, T, STEP>(ctx, b, pl, count, coefs, steps, o, XP, XT, XTn, A, Bm, parts);
}

static char const *muon_check(dlmi_newton_schulz const *ns) {
  if (ns == nullptr) return "null pointer";
  if (ns->steps < 1 || ns->steps > 64) return "1 to 64 steps";
  if (!(ns->eps >= 0.0f)) return "eps must not be negative";
  float const c[3] = {ns->a, ns->b, ns->c};
  if (!(muon_reach(c, ns->steps) <= 8.0)) return "coefficients that take singular values of [0, 1] out of the range the iteration is held in";
  return nullptr;
}

// Scratch that the matrices of one launch may take together.
constexpr size_t kMuonBudget = size_t(2) << 30;

static unsigned muon_group(MuonPlan const &pl, size_t left) {
  size_t n = kMuonBudget / pl.per_matrix;
  if (n < 1) n = 1;
  if (n > kMuonMax) n = kMuonMax;
  return static_cast<unsigned>(n < left ? n : left);
}

}  // namespace dlmi

using namespace dlmi;

extern "C" {

int dlmi_orthogonalize(dlmi_ctx *ctx, dlmi_dtype type, size_t rows, size_t cols, void const *G, void *O, dlmi_newton_schulz const *ns) {
  if (ctx == nullptr) return DLMI_E_INVALID;
  DLMI_REQUIRE(ctx, type == DLMI_F32 || type == DLMI_BF16, "unknown type");
  char const *const wrong = muon_check(ns);
  DLMI_REQUIRE(ctx, wrong == nullptr, wrong);
  DLMI_REQUIRE(ctx, rows <= DLMI_MUON_MAX_SIDE && cols <= DLMI_MUON_MAX_SIDE, "matrix too large");
  if (rows * cols == 0) return DLMI_OK;
  DLMI_REQUIRE_DEVICE(ctx);
  DLMI_REQUIRE(ctx, G != nullptr && O != nullptr, "null pointer");
  MuonBatch b = {};
  b.p[0] = O;
  b.g[0] = const_cast<void *>(G);
  float const c[3] = {ns->a, ns->b, ns->c};
  MuonPlan const pl = muon_plan(ctx, rows, cols, 1);
  int const rc = dlmi_scratch_reserve(ctx, pl.bytes(1));
  if (rc != DLMI_OK) return rc;
  if (type == DLMI_F32) return muon_batch<float, false>(ctx, b, rows, cols, 1, pl, 0.0f, 0, 0.0f, ns->steps, c, ns->eps);
  return muon_batch<__bf16, false>(ctx, b, rows, cols, 1, pl, 0.0f, 0, 0.0f, ns->steps, c, ns->eps);
}

int dlmi_opt_muon(dlmi_ctx *ctx, size_t n, dlmi_muon_problem const *problems, float momentum, int nesterov, float wd,
                  dlmi_newton_schulz const *ns) try {
  if (ctx == nullptr) return DLMI_E_INVALID;
  DLMI_REQUIRE(ctx, n == 0 || problems != nullptr, "null pointer");
  char const *const wrong = muon_check(ns);
  DLMI_REQUIRE(ctx, wrong == nullptr, wrong);
  if (n == 0) return DLMI_OK;
  DLMI_REQUIRE_DEVICE(ctx);
  // every array is updated in place, so none may be named twice
  struct Range {
    uintptr_t from, to;
  };
  std::vector<Range> ranges;
  for (size_t i = 0; i < n; ++i) {
    dlmi_muon_problem const &q = problems[i];
    DLMI_REQUIRE(ctx, q.rows <= DLMI_MUON_MAX_SIDE && q.cols <= DLMI_MUON_MAX_SIDE, "matrix too large");
    size_t const bytes = q.rows * q.cols * sizeof(float);
    if (bytes == 0) continue;
    DLMI_REQUIRE(ctx, q.params != nullptr && q.grads != nullptr && q.momentum != nullptr, "null pointer");
    for (float const *a : {q.params, q.grads, q.momentum})
      ranges.push_back({reinterpret_cast<uintptr_t>(a), reinterpret_cast<uintptr_t>(a) + bytes});
  }
  std::sort(ranges.begin(), ranges.end(), [](Range const &x, Range const &y) { return x.from < y.from; });
  for (size_t i = 1; i < ranges.size(); ++i) DLMI_REQUIRE(ctx, ranges[i].from >= ranges[i - 1].to, "two of the arrays overlap");
  // the launches and the scratch that the largest needs are settled before the first array is touched
  struct Launch {
    MuonBatch b;
    MuonPlan pl;
    size_t rows, cols;
    unsigned count;
  };
  std::vector<Launch> launches;
  std::vector<char> done(n, 0);
  std::vector<size_t> same;
  size_t scratch = 0;
  for (size_t i = 0; i < n; ++i) {
    size_t const rows = problems[i].rows, cols = problems[i].cols;
    if (done[i] || rows * cols == 0) continue;
    same.clear();
    for (size_t k = i; k < n; ++k)
      if (!done[k] && problems[k].rows == rows && problems[k].cols == cols) {
        same.push_back(k);
        done[k] = 1;
      }
    for (size_t at = 0; at < same.size();) {
      size_t const left = same.size() - at;
      Launch l = {};
      l.pl = muon_plan(ctx, rows, cols, left < kMuonMax ? left : kMuonMax);
      l.rows = rows;
      l.cols = cols;
      l.count = muon_group(l.pl, left);
      for (unsigned k = 0; k < l.count; ++k) {
        dlmi_muon_problem const &q = problems[same[at + k]];
        l.b.p[k] = q.params;
        l.b.g[k] = q.grads;
        l.b.m[k] = q.momentum;
        l.b.lr[k] = q.lr;
      }
      if (l.pl.bytes(l.count) > scratch) scratch = l.pl.bytes(l.count);
      at += l.count;
      launches.push_back(l);
    }
  }
  int rc = scratch != 0 ? dlmi_scratch_reserve(ctx, scratch) : DLMI_OK;
  float const c[3] = {ns->a, ns->b, ns->c};
  for (size_t i = 0; rc == DLMI_OK && i < launches.size(); ++i) {
    Launch const &l = launches[i];
    rc = muon_batch<float, true>(ctx, l.b, l.rows, l.cols, l.count, l.pl, momentum, nesterov, wd, ns->steps, c, ns->eps);
  }
  return rc;
} catch (std::bad_alloc const &) {
  return dlmi_fail(ctx, DLMI_E_NOMEM, "dlmi_opt_muon: out of host memory");
}

}  // extern "C"
