// The tail of a residual block with row norms, fused, for gfx950:
//
//   y = rs x + bs f(gate) post(u)      the block's output u normalized, gated, scaled and added to the stream x
//   h = pre(y)                         the next block's input
//
// and its gradient.  post and pre are nothing, v / rms(v) or (v - mean(v)) / std(v) over a row (eps under the root), times
// a weight, plus a bias; f is the identity, the sigmoid or tanh; gate_rows consecutive rows share a row of the gate.
//
// With t = dy + (pre's gradient of dh at y) and dn = bs t f(gate):
//   dx = rs t;  du = (post's gradient of dn at u);  dgate = sum over the rows that share it of bs t f'(gate) post(u)
//   a norm v^ = (v - m) r w: dv = r (g - [mean g] - v^ mean(g v^)), g = d w (the bracket for the layer norm alone)
//   dw = sum over rows of d v^, db = sum over rows of d
//
// Bound by memory: a row is read once into registers, every statistic is taken there (the variance from centred values)
// and every output leaves once; forward 4 tensors, backward 6 (plus the gate and its gradient).  A workgroup keeps a
// row's columns on the same threads over all its rows, so weights are read once per workgroup and the column sums of the
// backward stay in registers: one partial row per workgroup, added in a fixed order by a second launch (no atomics:
// the same bits every time).  Nothing is kept from the forward but y: the statistics are formed again from u and y.
#include "dlmi_common.hpp"

namespace dlmi {

constexpr int kBnMaxWidth = DLMI_BLOCK_NORM_MAX_WIDTH;

typedef float f32x4v __attribute__((ext_vector_type(4)));

// N consecutive columns in one access, at any alignment (the hardware takes unaligned ones).
template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) BnVec {
  T v[N];
};

// The same for rows, which are read and written once: first to leave the caches.  [8192 x 4096] FP32 forward 124 -> 112 us =
// 6.0 TB/s (stores alone: 120 us), [16384 x 4096] BF16 backward 191 -> 174 us = 4.6 TB/s; a copy of 1 GiB runs at 5.1 TB/s.
typedef unsigned BnWords __attribute__((ext_vector_type(4), aligned(2)));
template <class T, int N>
__device__ __forceinline__ BnVec<T, N> bn_read(T const *p) {
  if constexpr (sizeof(BnVec<T, N>) == 16) {
    BnWords const w = __builtin_nontemporal_load(reinterpret_cast<BnWords const *>(p));
    return __builtin_bit_cast(BnVec<T, N>, w);
  } else {
    return *reinterpret_cast<BnVec<T, N> const *>(p);
  }
}
template <class T, int N>
__device__ __forceinline__ void bn_write(T *p, BnVec<T, N> const &v) {
  if constexpr (sizeof(BnVec<T, N>) == 16)
    __builtin_nontemporal_store(__builtin_bit_cast(BnWords, v), reinterpret_cast<BnWords *>(p));
  else
    *reinterpret_cast<BnVec<T, N> *>(p) = v;
}

// A thread's pieces of a row: C of them, N columns each, NT * N apart.  A piece that hangs over the row's end is moved back
// to end with it, and its first `shift` columns, which belong to the thread before, are left alone: all loads are whole and
// without conditions, which the compiler would wait behind (rows prefetched behind branches: 154 us against 129 us at
// [8192 x 4096] FP32 forward).  H >= N.
template <int N, int NT, int C>
struct BnPlace {
  int pos[C], shift[C];
  bool tail;  // this wavefront has such a piece
  __device__ __forceinline__ explicit BnPlace(int H) {
    bool t = false;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      int const col = (c * NT + static_cast<int>(threadIdx.x)) * N;
      pos[c] = col < H - N ? col : H - N;
      shift[c] = col - pos[c];
      t = t || shift[c] != 0;
    }
    tail = __any(t);
  }
};

template <class T, int N, int C>
struct BnRaw {
  BnVec<T, N> v[C];
};

template <class T, int N, int NT, int C>
__device__ __forceinline__ void bn_fetch(BnRaw<T, N, C> &o, T const *row, BnPlace<N, NT, C> const &at) {
#pragma unroll
  for (int c = 0; c < C; ++c) o.v[c] = bn_read<T, N>(row + at.pos[c]);
}
template <class T, int N, int NT, int C>
__device__ __forceinline__ void bn_widen(float (&o)[C][N], BnRaw<T, N, C> const &r, BnPlace<N, NT, C> const &at) {
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < N; ++i) o[c][i] = static_cast<float>(r.v[c].v[i]);
  if (at.tail) {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < N; ++i) o[c][i] = i >= at.shift[c] ? o[c][i] : 0.0f;
  }
}
template <class T, int N, int NT, int C>
__device__ __forceinline__ void bn_store(T *row, float const (&o)[C][N], BnPlace<N, NT, C> const &at) {
#pragma unroll
  for (int c = 0; c < C; ++c) {
    BnVec<T, N> v;
#pragma unroll
    for (int i = 0; i < N; ++i) v.v[i] = static_cast<T>(o[c][i]);
    if (at.shift[c] == 0) {
      bn_write<T, N>(row + at.pos[c], v);
    } else {
#pragma unroll
      for (int i = 1; i < N; ++i)
        if (i >= at.shift[c]) row[at.pos[c] + i] = v.v[i];
    }
  }
}
template <int N, int NT, int C>
__device__ __forceinline__ void bn_param(float const *p, float dflt, float (&o)[C][N], BnPlace<N, NT, C> const &at) {
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < N; ++i) o[c][i] = dflt;
  if (p == nullptr) return;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    BnVec<float, N> const v = *reinterpret_cast<BnVec<float, N> const *>(p + at.pos[c]);
#pragma unroll
    for (int i = 0; i < N; ++i) o[c][i] = v.v[i];
  }
}

// Sum over each 16 lanes, the same in all of them (DPP).
__device__ __forceinline__ float bn_row_sum(float v) {
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xf, 0xf, false));   // lane ^ 1
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xf, 0xf, false));   // lane ^ 2
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xf, 0xf, false));  // mirrored in 8
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xf, 0xf, false));  // mirrored in 16
  return v;
}
// Over the 64 lanes, without LDS: rows of 16 and halves are swapped.
__device__ __forceinline__ float bn_wave_sum(float v) {
  v = bn_row_sum(v);
  unsigned const r = __float_as_uint(v);
  auto const p = __builtin_amdgcn_permlane16_swap(r, r, false, false);
  v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  unsigned const h = __float_as_uint(v);
  auto const q = __builtin_amdgcn_permlane32_swap(h, h, false, false);
  return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}

// Sums of K values over the NT threads of a row, the same in every thread.  Consecutive sums use alternating halves of
// `lds` (flip), so one barrier each is enough: who writes a half again has passed the barrier behind its last reading.
template <int NT, int K>
__device__ __forceinline__ void bn_sums(float (&v)[K], float (*lds)[16][4], int &flip) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = bn_wave_sum(v[k]);
  if constexpr (NT > 64) {
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) lds[flip][threadIdx.x >> 6][k] = v[k];
    }
    __syncthreads();
    // a row of 16 lanes takes the wavefronts' shares, one each
    int const w = threadIdx.x & 15;
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = bn_row_sum(w < NT / 64 ? lds[flip][w][k] : 0.0f);
    flip ^= 1;
  }
}

// tanh near 0 by its Taylor series (the next term is below 5e-8 of it), where 1 - e of the quotient cancels.
__device__ __forceinline__ float bn_gate(int act, float g) {
  if (act == DLMI_ACT_SIGMOID) return __builtin_amdgcn_rcpf(1.0f + __expf(-g));
  if (act == DLMI_ACT_TANH) {
    float const m = fabsf(g), e = __expf(-2.0f * m), q = g * g;
    float const far = copysignf((1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e), g);
    float const near = g + g * q * (-1.0f / 3.0f + q * (2.0f / 15.0f + q * (-17.0f / 315.0f + q * (62.0f / 2835.0f))));
    return m < 0.3f ? near : far;
  }
  return g;
}
__device__ __forceinline__ float bn_gate_slope(int act, float f) {
  if (act == DLMI_ACT_SIGMOID) return f * (1.0f - f);
  if (act == DLMI_ACT_TANH) return 1.0f - f * f;
  return 1.0f;
}

struct BnArgs {
  void const *x, *u, *gate;
  float const *w_post, *b_post, *w_pre, *b_pre;
  void *y, *h;
  // backward
  void const *dy, *dh;
  void *dx, *du, *dgate;
  float *partial;       // [workgroups][planes][H]
  int plane[5];         // of dw_post, db_post, dw_pre, db_pre, the shared gate; -1: not asked for
  int planes;
  int direct;           // a workgroup covers whole runs of rows that share a gate: it writes dgate itself
  size_t B;
  int H;
  int post, pre, act;
  size_t gate_rows;     // 0: no gate
  size_t rows_per_wg;   // direct: rows of a workgroup (a multiple of gate_rows); otherwise rows of a slice
  unsigned slices;      // of a run of gate_rows rows
  float rs, bs, eps_post, eps_pre;
};

#define BN_EACH                     \
  _Pragma("unroll") for (int c = 0; c < C; ++c) _Pragma("unroll") for (int i = 0; i < N; ++i)
#define BN_IN (i >= at_.shift[c])

template <class T, int N, int NT, int C>
__global__ __launch_bounds__(NT) void k_block_norm_fwd(BnArgs a) {
  __shared__ float lds[2][16][4];
  int flip = 0;
  int const H = a.H;
  float const inv_h = 1.0f / static_cast<float>(H);
  BnPlace<N, NT, C> const at_(H);
  BnRaw<T, N, C> ru, rx, rg;
  auto const fetch = [&](size_t r) {
    size_t const at = r * static_cast<size_t>(H);
    bn_fetch(ru, static_cast<T const *>(a.u) + at, at_);
    bn_fetch(rx, static_cast<T const *>(a.x) + at, at_);
    if (a.gate_rows != 0) bn_fetch(rg, static_cast<T const *>(a.gate) + (a.gate_rows == 1 ? r : r / a.gate_rows) * static_cast<size_t>(H), at_);
  };
  if (blockIdx.x < a.B) fetch(blockIdx.x);
  float w1[C][N], b1[C][N], w2[C][N], b2[C][N];
  bn_param(a.w_post, 1.0f, w1, at_);
  bn_param(a.b_post, 0.0f, b1, at_);
  bn_param(a.w_pre, 1.0f, w2, at_);
  bn_param(a.b_pre, 0.0f, b2, at_);
  // the columns that are another thread's are zero; what centring makes of them stays out of the sums
  auto const norm = [&](float (&v)[C][N], int how, float eps) {
    if (how == DLMI_ROW_NORM_NONE) return;
    if (how == DLMI_ROW_NORM_LAYER) {
      float s[1] = {0.0f};
      BN_EACH s[0] += v[c][i];
      bn_sums<NT>(s, lds, flip);
      float const mean = s[0] * inv_h;
      BN_EACH v[c][i] = BN_IN ? v[c][i] - mean : 0.0f;
    }
    float q[1] = {0.0f};
    BN_EACH q[0] += v[c][i] * v[c][i];
    bn_sums<NT>(q, lds, flip);
    float const rstd = 1.0f / sqrtf(q[0] * inv_h + eps);
    BN_EACH v[c][i] *= rstd;
  };
  for (size_t r = blockIdx.x; r < a.B; r += gridDim.x) {
    size_t const at = r * static_cast<size_t>(H);
    float u[C][N], x[C][N], g[C][N];
    bn_widen(u, ru, at_);
    bn_widen(x, rx, at_);
    if (a.gate_rows != 0) bn_widen(g, rg, at_);
    // the next row is on its way while this one is worked on (y may be x and h may be u: this row's only)
    if (r + gridDim.x < a.B) fetch(r + gridDim.x);
    norm(u, a.post, a.eps_post);
    BN_EACH {
      float n = u[c][i] * w1[c][i] + b1[c][i];
      if (a.gate_rows != 0) n *= bn_gate(a.act, g[c][i]);
      x[c][i] = a.rs * x[c][i] + a.bs * n;
    }
    bn_store(static_cast<T *>(a.y) + at, x, at_);
    BN_EACH x[c][i] = BN_IN ? x[c][i] : 0.0f;
    norm(x, a.pre, a.eps_pre);
    BN_EACH x[c][i] = x[c][i] * w2[c][i] + b2[c][i];
    bn_store(static_cast<T *>(a.h) + at, x, at_);
  }
}

enum { kBnNoGate = 0, kBnGateEach = 1, kBnGateShared = 2 };

// GATE: none, one row each, or shared by rows (f is formed once per run then, and its slope multiplies the finished sum).
// BIAS: post has a bias, or a bias's gradient is asked for.
// A thread keeps its columns' sums and the row at hand and the next in registers; the weights (and a shared gate's f) it
// reads again every row from LDS, which only it uses: with them in registers too, two workgroups of 8 wavefronts did not
// fit a CU without spilling ([16384 x 4096] bf16, shared gate: 511 us then).
template <class T, int N, int NT, int C, int GATE, bool BIAS>
__global__ __launch_bounds__(NT, NT <= 512 && C * N <= 8 ? 4 : 1) void k_block_norm_bwd(BnArgs a) {
  constexpr int Q = N >= 4 ? C * N / 4 : 1;
  constexpr bool kLds = N >= 4 && C * N <= 8;  // wider rows (and those of a few columns) read the weights from memory
  __shared__ float lds[2][16][4];
  __shared__ f32x4v kept[kLds ? 2 + (BIAS ? 1 : 0) + (GATE == kBnGateShared ? 1 : 0) : 1][kLds ? Q : 1][kLds ? NT : 1];
  constexpr int kW1 = 0, kW2 = 1, kF = 2, kB1 = GATE == kBnGateShared ? 3 : 2;
  int flip = 0;
  int const H = a.H;
  float const inv_h = 1.0f / static_cast<float>(H);
  BnPlace<N, NT, C> const at_(H);
  auto const keep = [&](int k, float const (&v)[C][N]) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      f32x4v x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = v[(q * 4 + j) / N][(q * 4 + j) % N];
      kept[k][q][threadIdx.x] = x;
    }
  };
  auto const back = [&](int k, float (&v)[C][N]) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      f32x4v const x = kept[k][q][threadIdx.x];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[(q * 4 + j) / N][(q * 4 + j) % N] = x[j];
    }
  };
  auto const params = [&](float const *p, float dflt, float (&v)[C][N]) { bn_param(p, dflt, v, at_); };
  size_t r0, r1;
  if (a.direct) {
    r0 = blockIdx.x * a.rows_per_wg;
    r1 = r0 + a.rows_per_wg;
  } else {
    size_t const run = blockIdx.x / a.slices;
    r0 = run * a.gate_rows + (blockIdx.x % a.slices) * a.rows_per_wg;
    r1 = r0 + a.rows_per_wg;
    if (r1 > (run + 1) * a.gate_rows) r1 = (run + 1) * a.gate_rows;
  }
  if (r1 > a.B) r1 = a.B;
  bool const live_y = a.dh != nullptr && a.pre != DLMI_ROW_NORM_NONE;
  BnRaw<T, N, C> ru, ry, rt, re, rg;
  auto const fetch = [&](size_t r) {
    size_t const at = r * static_cast<size_t>(H);
    bn_fetch(ru, static_cast<T const *>(a.u) + at, at_);
    if (live_y) bn_fetch(ry, static_cast<T const *>(a.y) + at, at_);
    if (a.dy != nullptr) bn_fetch(rt, static_cast<T const *>(a.dy) + at, at_);
    if (a.dh != nullptr) bn_fetch(re, static_cast<T const *>(a.dh) + at, at_);
    if constexpr (GATE == kBnGateEach) bn_fetch(rg, static_cast<T const *>(a.gate) + at, at_);
  };
  if (r0 < r1) fetch(r0);
  if constexpr (kLds) {
    float v[C][N];
    params(a.w_post, 1.0f, v);
    keep(kW1, v);
    params(a.w_pre, 1.0f, v);
    keep(kW2, v);
    if constexpr (BIAS) {
      params(a.b_post, 0.0f, v);
      keep(kB1, v);
    }
  }
  // the weights and the shared gate of this thread's columns, for the moment
  auto const weight = [&](int k, float (&v)[C][N]) {
    if constexpr (kLds)
      back(k, v);
    else
      params(k == kW1 ? a.w_post : a.w_pre, 1.0f, v);
  };
  auto const bias = [&](float (&v)[C][N]) {
    if constexpr (kLds)
      back(kB1, v);
    else
      params(a.b_post, 0.0f, v);
  };
  auto const gate_row = [&](size_t r, float (&v)[C][N]) {
    bn_fetch(rg, static_cast<T const *>(a.gate) + r / a.gate_rows * static_cast<size_t>(H), at_);
    bn_widen(v, rg, at_);
    BN_EACH v[c][i] = bn_gate(a.act, v[c][i]);
  };
  auto const shared_gate = [&](size_t r, float (&v)[C][N]) {
    if constexpr (kLds)
      back(kF, v);
    else
      gate_row(r, v);
  };
  float dw1[C][N], db1[C][N], dw2[C][N], db2[C][N], dg[C][N];
  BN_EACH dw1[c][i] = db1[c][i] = dw2[c][i] = db2[c][i] = dg[c][i] = 0.0f;
  for (size_t r = r0; r < r1; ++r) {
    size_t const at = r * static_cast<size_t>(H);
    float u[C][N], y[C][N], t[C][N], e[C][N];
    bn_widen(u, ru, at_);
    if (live_y) bn_widen(y, ry, at_);
    if (a.dy != nullptr)
      bn_widen(t, rt, at_);
    else
      BN_EACH t[c][i] = 0.0f;
    if (a.dh != nullptr)
      bn_widen(e, re, at_);
    else
      BN_EACH e[c][i] = 0.0f;
    BnRaw<T, N, C> rgr;
    if constexpr (GATE == kBnGateEach) rgr = rg;
    if constexpr (GATE == kBnGateShared && kLds) {
      if (r == r0 || r % a.gate_rows == 0) {
        float v[C][N];
        gate_row(r, v);
        keep(kF, v);
      }
    }
    // the next row is on its way while this one is worked on (dx may be dy and du may be dh: this row's only)
    if (r + 1 < r1) fetch(r + 1);
    // the means, where a layer norm asks for them
    if (a.post == DLMI_ROW_NORM_LAYER || (live_y && a.pre == DLMI_ROW_NORM_LAYER)) {
      float s[2] = {0.0f, 0.0f};
      BN_EACH {
        s[0] += u[c][i];
        if (live_y) s[1] += y[c][i];
      }
      bn_sums<NT>(s, lds, flip);
      float const mu = a.post == DLMI_ROW_NORM_LAYER ? s[0] * inv_h : 0.0f;
      float const my = a.pre == DLMI_ROW_NORM_LAYER ? s[1] * inv_h : 0.0f;
      BN_EACH {
        u[c][i] = BN_IN ? u[c][i] - mu : 0.0f;
        if (live_y) y[c][i] = BN_IN ? y[c][i] - my : 0.0f;
      }
    }
    // pre's gradient
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    float w[C][N];
    if (live_y) weight(kW2, w);
    BN_EACH {
      s[0] += u[c][i] * u[c][i];
      if (live_y) {
        float const gh = e[c][i] * w[c][i];
        s[1] += y[c][i] * y[c][i];
        s[2] += gh;
        s[3] += gh * y[c][i];
      }
    }
    bn_sums<NT>(s, lds, flip);
    float const ru_ = a.post != DLMI_ROW_NORM_NONE ? 1.0f / sqrtf(s[0] * inv_h + a.eps_post) : 1.0f;
    if (live_y) {
      float const ry_ = 1.0f / sqrtf(s[1] * inv_h + a.eps_pre);
      float const c1 = a.pre == DLMI_ROW_NORM_LAYER ? s[2] * inv_h : 0.0f;
      float const c2 = s[3] * ry_ * inv_h;
      weight(kW2, w);
      BN_EACH {
        float const yh = y[c][i] * ry_;
        dw2[c][i] += e[c][i] * yh;
        if constexpr (BIAS) db2[c][i] += e[c][i];
        t[c][i] += ry_ * (e[c][i] * w[c][i] - c1 - yh * c2);
      }
    } else {
      BN_EACH t[c][i] += e[c][i];
    }
    // the gate, then post's gradient; e becomes dn
    float p[2] = {0.0f, 0.0f};
    float f[C][N], b1[C][N];
    weight(kW1, w);
    if constexpr (GATE == kBnGateEach) {
      bn_widen(f, rgr, at_);
      BN_EACH f[c][i] = bn_gate(a.act, f[c][i]);
    }
    if constexpr (GATE == kBnGateShared) shared_gate(r, f);
    if constexpr (BIAS && GATE != kBnNoGate) bias(b1);
    BN_EACH {
      float const uh = u[c][i] * ru_;
      float d = BN_IN ? a.bs * t[c][i] : 0.0f;
      if constexpr (GATE != kBnNoGate) {
        float n = uh * w[c][i];
        if constexpr (BIAS) n += b1[c][i];
        if constexpr (GATE == kBnGateEach)
          dg[c][i] = d * bn_gate_slope(a.act, f[c][i]) * n;
        else
          dg[c][i] += d * n;
        d *= f[c][i];
      }
      dw1[c][i] += d * uh;
      if constexpr (BIAS) db1[c][i] += d;
      float const gd = d * w[c][i];
      p[0] += gd;
      p[1] += gd * uh;
      e[c][i] = d;
      t[c][i] *= a.rs;
      u[c][i] = uh;
    }
    bn_store(static_cast<T *>(a.dx) + at, t, at_);
    if (a.post != DLMI_ROW_NORM_NONE) {
      bn_sums<NT>(p, lds, flip);
      weight(kW1, w);
      float const c1 = a.post == DLMI_ROW_NORM_LAYER ? p[0] * inv_h : 0.0f, c2 = p[1] * inv_h;
      BN_EACH e[c][i] = ru_ * (e[c][i] * w[c][i] - c1 - u[c][i] * c2);
    }
    bn_store(static_cast<T *>(a.du) + at, e, at_);
    if constexpr (GATE == kBnGateEach) {
      if (a.dgate != nullptr) bn_store(static_cast<T *>(a.dgate) + at, dg, at_);
    }
    if constexpr (GATE == kBnGateShared) {
      if (a.direct && ((r + 1) % a.gate_rows == 0 || r + 1 == a.B)) {
        shared_gate(r, f);
        BN_EACH dg[c][i] *= bn_gate_slope(a.act, f[c][i]);
        if (a.dgate != nullptr) {
          T *const out = static_cast<T *>(a.dgate) + r / a.gate_rows * static_cast<size_t>(H);
          bn_store(out, dg, at_);
        }
        BN_EACH dg[c][i] = 0.0f;
      }
    }
  }
  if (a.partial == nullptr) return;
  float *const out = a.partial + static_cast<size_t>(blockIdx.x) * a.planes * H;
  auto const leave = [&](int plane, float const (&v)[C][N]) {
    if (plane < 0) return;
    bn_store(out + static_cast<size_t>(plane) * H, v, at_);
  };
  leave(a.plane[0], dw1);
  if constexpr (BIAS) leave(a.plane[1], db1);
  leave(a.plane[2], dw2);
  if constexpr (BIAS) leave(a.plane[3], db2);
  if constexpr (GATE == kBnGateShared) {
    if (r0 < r1) {
      float f[C][N];
      shared_gate(r1 - 1, f);
      BN_EACH dg[c][i] *= bn_gate_slope(a.act, f[c][i]);
    }
    leave(a.plane[4], dg);
  }
}

struct BnReduce {
  float const *partial;
  int plane[5], planes;
  float *out[4];      // the parameters' gradients
  void *dgate;        // [runs][H]
  unsigned workgroups, slices;
  int H, accumulate;
};

// 64 columns of one plane: 16 threads per column add every 16th row, then a tree.  blockIdx.y: a plane of the parameters'
// gradients (over all workgroups), from `params` on a run's slices of the gate's.
template <class T>
__global__ __launch_bounds__(1024) void k_block_norm_reduce(BnReduce a, unsigned params) {
  __shared__ float lds[16][64];
  bool const gate = blockIdx.y >= params;
  int which = 4;
  if (!gate)
    for (which = 0; a.plane[which] != static_cast<int>(blockIdx.y); ++which) {
    }
  int const plane = a.plane[which];
  unsigned const from = gate ? (blockIdx.y - params) * a.slices : 0, n = gate ? a.slices : a.workgroups;
  int const col = static_cast<int>(blockIdx.x * 64 + (threadIdx.x & 63));
  unsigned const part = threadIdx.x >> 6;
  float s = 0.0f;
  if (col < a.H) {
    float const *const p = a.partial + static_cast<size_t>(plane) * a.H + col;
    size_t const step = static_cast<size_t>(a.planes) * a.H;
#pragma unroll 8
    for (unsigned w = part; w < n; w += 16) s += p[(from + w) * step];
  }
  lds[part][threadIdx.x & 63] = s;
  __syncthreads();
  for (unsigned o = 8; o > 0; o >>= 1) {
    if (part < o) lds[part][threadIdx.x & 63] += lds[part + o][threadIdx.x & 63];
    __syncthreads();
  }
  if (part != 0 || col >= a.H) return;
  s = lds[0][threadIdx.x & 63];
  if (!gate)
    a.out[which][col] = a.accumulate ? a.out[which][col] + s : s;
  else
    static_cast<T *>(a.dgate)[static_cast<size_t>(blockIdx.y - params) * a.H + col] = static_cast<T>(s);
}

template <class T, int N, int NT, int C, int GATE>
static void bn_launch_bwd(dlmi_ctx *ctx, BnArgs const &a, unsigned blocks) {
  if (a.b_post != nullptr || a.plane[1] >= 0 || a.plane[3] >= 0)
    hipLaunchKernelGGL((k_block_norm_bwd<T, N, NT, C, GATE, true>), dim3(blocks), dim3(NT), 0, ctx->stream, a);
  else
    hipLaunchKernelGGL((k_block_norm_bwd<T, N, NT, C, GATE, false>), dim3(blocks), dim3(NT), 0, ctx->stream, a);
}

template <class T, int N, int NT, int C, bool BACK>
static void bn_launch(dlmi_ctx *ctx, BnArgs const &a, unsigned blocks) {
  if constexpr (!BACK)
    hipLaunchKernelGGL((k_block_norm_fwd<T, N, NT, C>), dim3(blocks), dim3(NT), 0, ctx->stream, a);
  else if (a.gate_rows == 0)
    bn_launch_bwd<T, N, NT, C, kBnNoGate>(ctx, a, blocks);
  else if (a.gate_rows == 1)
    bn_launch_bwd<T, N, NT, C, kBnGateEach>(ctx, a, blocks);
  else
    bn_launch_bwd<T, N, NT, C, kBnGateShared>(ctx, a, blocks);
}

// Threads of a row: `each` columns each, up to 1024 threads.
static int bn_threads(int H, int each) {
  int nt = 64;
  while (nt < 1024 && nt * each < H) nt *= 2;
  return nt;
}
// Columns of a thread: 8, but 4 in the fp32 backward, whose rows at hand and next take twice the registers of bf16's (with 8
// they spilled).  Rows wider than 1024 threads of these take two or four times as many.
static int bn_each(dlmi_dtype type, bool back) { return back && type == DLMI_F32 ? 4 : 8; }

template <class T, int C, bool BACK>
static void bn_dispatch_each(dlmi_ctx *ctx, BnArgs const &a, unsigned blocks) {
  constexpr int N = 16 / static_cast<int>(sizeof(T));  // 16-byte accesses
  if (a.H < N) return bn_launch<T, 1, 64, 1, BACK>(ctx, a, blocks);
  switch (bn_threads(a.H, C * N)) {
    case 64: return bn_launch<T, N, 64, C, BACK>(ctx, a, blocks);
    case 128: return bn_launch<T, N, 128, C, BACK>(ctx, a, blocks);
    case 256: return bn_launch<T, N, 256, C, BACK>(ctx, a, blocks);
    case 512: return bn_launch<T, N, 512, C, BACK>(ctx, a, blocks);
    default: break;
  }
  if (a.H <= 1024 * C * N) return bn_launch<T, N, 1024, C, BACK>(ctx, a, blocks);
  if constexpr (C * N < 8) {
    if (a.H <= 8192) return bn_launch<T, N, 1024, 8 / N, BACK>(ctx, a, blocks);
  }
  return bn_launch<T, N, 1024, 16 / N, BACK>(ctx, a, blocks);
}

static void bn_dispatch(dlmi_ctx *ctx, dlmi_dtype type, bool back, BnArgs const &a, unsigned blocks) {
  if (type == DLMI_BF16 && back)
    bn_dispatch_each<__bf16, 1, true>(ctx, a, blocks);
  else if (type == DLMI_BF16)
    bn_dispatch_each<__bf16, 1, false>(ctx, a, blocks);
  else if (back)
    bn_dispatch_each<float, 1, true>(ctx, a, blocks);
  else
    bn_dispatch_each<float, 2, false>(ctx, a, blocks);
}

static char const *bn_check(dlmi_block_norm_desc const *d, size_t B, size_t H, void const *gate, float const *w_post,
                            float const *b_post, float const *w_pre, float const *b_pre) {
  if (d == nullptr) return "null descriptor";
  auto const known = [](dlmi_row_norm n) { return n == DLMI_ROW_NORM_NONE || n == DLMI_ROW_NORM_RMS || n == DLMI_ROW_NORM_LAYER; };
  if (!known(d->post) || !known(d->pre)) return "unknown norm";
  if (d->gate_rows != 0 && gate == nullptr) return "gate_rows without a gate";
  if (d->gate_rows == 0 && gate != nullptr) return "a gate without gate_rows";
  if (d->gate_act != DLMI_ACT_LINEAR && d->gate_act != DLMI_ACT_SIGMOID && d->gate_act != DLMI_ACT_TANH)
    return "the gate's activation must be linear, sigmoid or tanh";
  if (d->post == DLMI_ROW_NORM_NONE && (w_post != nullptr || b_post != nullptr)) return "weight or bias without a norm after the block";
  if (d->pre == DLMI_ROW_NORM_NONE && (w_pre != nullptr || b_pre != nullptr)) return "weight or bias without a norm before the block";
  if (!(d->eps_post >= 0.0f) || !(d->eps_pre >= 0.0f)) return "eps must not be negative";
  if (B > 0x7fffffffu) return "too many rows";
  return nullptr;
}

static BnArgs bn_args(dlmi_block_norm_desc const *d, size_t B, size_t H) {
  BnArgs a = {};
  a.B = B;
  a.H = static_cast<int>(H);
  a.post = d->post;
  a.pre = d->pre;
  a.act = d->gate_act;
  a.gate_rows = d->gate_rows < B ? d->gate_rows : B;  // one row for all, whatever lies beyond
  a.rs = d->residual_scale;
  a.bs = d->branch_scale;
  a.eps_post = d->eps_post;
  a.eps_pre = d->eps_pre;
  return a;
}

// No rows: sums over none of them.
static int bn_no_rows(dlmi_ctx *ctx, size_t B, size_t H, float *dw_post, float *db_post, float *dw_pre, float *db_pre, int accumulate) {
  if (B != 0 || H == 0 || accumulate) return DLMI_OK;
  DLMI_REQUIRE_DEVICE(ctx);
  BnReduce r = {};
  float *const params[4] = {dw_post, db_post, dw_pre, db_pre};
  unsigned sums = 0;
  for (int k = 0; k < 4; ++k) {
    r.plane[k] = params[k] != nullptr ? static_cast<int>(sums++) : -1;
    r.out[k] = params[k];
  }
  if (sums == 0) return DLMI_OK;
  r.H = static_cast<int>(H);
  hipLaunchKernelGGL(k_block_norm_reduce<float>, dim3(static_cast<unsigned>(dlmi_ceil_div(H, 64)), sums), dim3(1024), 0, ctx->stream, r, sums);
  DLMI_LAUNCH_CHECK(ctx, "k_block_norm_reduce");
  return DLMI_OK;
}

}  // namespace dlmi

using namespace dlmi;

extern "C" {

int dlmi_block_norm_fwd(dlmi_ctx *ctx, dlmi_dtype type, dlmi_block_norm_desc const *desc, size_t B, size_t H, void const *x,
                        void const *u, void const *gate, float const *w_post, float const *b_post, float const *w_pre,
                        float const *b_pre, void *y, void *h) {
  if (ctx == nullptr) return DLMI_E_INVALID;
  DLMI_REQUIRE(ctx, type == DLMI_F32 || type == DLMI_BF16, "unknown type");
  char const *const wrong = bn_check(desc, B, H, gate, w_post, b_post, w_pre, b_pre);
  DLMI_REQUIRE(ctx, wrong == nullptr, wrong);
  if (H > DLMI_BLOCK_NORM_MAX_WIDTH) return dlmi_fail(ctx, DLMI_E_UNSUPPORTED, "%s: rows wider than %d", __func__, kBnMaxWidth);
  if (B * H == 0) return DLMI_OK;
  DLMI_REQUIRE_DEVICE(ctx);
  DLMI_REQUIRE(ctx, x != nullptr && u != nullptr && y != nullptr && h != nullptr, "null pointer");
  size_t const row = H * (type == DLMI_F32 ? 4 : 2);
  BnArgs a = bn_args(desc, B, H);
  dlmi_span const spans[] = {{y, B * row, true},  {h, B * row, true},       {x, B * row, true},      {u, B * row, true},
                             {gate, a.gate_rows != 0 ? dlmi_ceil_div(B, a.gate_rows) * row : 0, false}, {w_post, H * 4, false},
                             {b_post, H * 4, false}, {w_pre, H * 4, false}, {b_pre, H * 4, false}};
  DLMI_REQUIRE(ctx, !dlmi_spans_collide(spans, 2, 9), "an output overlaps another array");
  a.x = x;
  a.u = u;
  a.gate = gate;
  a.w_post = w_post;
  a.b_post = b_post;
  a.w_pre = w_pre;
  a.b_pre = b_pre;
  a.y = y;
  a.h = h;
  size_t blocks = static_cast<size_t>(ctx->num_cu) * (2048 / bn_threads(a.H, bn_each(type, false)));
  if (blocks > B) blocks = B;
  bn_dispatch(ctx, type, false, a, static_cast<unsigned>(blocks));
  DLMI_LAUNCH_CHECK(ctx, "k_block_norm_fwd");
  return DLMI_OK;
}

int dlmi_block_norm_bwd(dlmi_ctx *ctx, dlmi_dtype type, dlmi_block_norm_desc const *desc, size_t B, size_t H, void const *u,
                        void const *y, void const *gate, float const *w_post, float const *b_post, float const *w_pre,
                        void const *dy, void const *dh, void *dx, void *du, void *dgate, float *dw_post, float *db_post,
                        float *dw_pre, float *db_pre, int accumulate) {
  if (ctx == nullptr) return DLMI_E_INVALID;
  DLMI_REQUIRE(ctx, type == DLMI_F32 || type == DLMI_BF16, "unknown type");
  char const *const wrong = bn_check(desc, B, H, gate, w_post, b_post, w_pre, nullptr);
  DLMI_REQUIRE(ctx, wrong == nullptr, wrong);
  DLMI_REQUIRE(ctx, desc->post != DLMI_ROW_NORM_NONE || (dw_post == nullptr && db_post == nullptr), "gradients of a norm after the block that is not there");
  DLMI_REQUIRE(ctx, desc->pre != DLMI_ROW_NORM_NONE || (dw_pre == nullptr && db_pre == nullptr), "gradients of a norm before the block that is not there");
  DLMI_REQUIRE(ctx, desc->gate_rows != 0 || dgate == nullptr, "the gradient of a gate that is not there");
  if (H > DLMI_BLOCK_NORM_MAX_WIDTH) return dlmi_fail(ctx, DLMI_E_UNSUPPORTED, "%s: rows wider than %d", __func__, kBnMaxWidth);
  if (B * H == 0) return bn_no_rows(ctx, B, H, dw_post, db_post, dw_pre, db_pre, accumulate);
  DLMI_REQUIRE_DEVICE(ctx);
  DLMI_REQUIRE(ctx, u != nullptr && dx != nullptr && du != nullptr, "null pointer");
  DLMI_REQUIRE(ctx, dy != nullptr || dh != nullptr, "no gradient to start from");
  DLMI_REQUIRE(ctx, y != nullptr || dh == nullptr || desc->pre == DLMI_ROW_NORM_NONE, "null pointer");
  BnArgs a = bn_args(desc, B, H);
  size_t const row = H * (type == DLMI_F32 ? 4 : 2);
  size_t const gr = a.gate_rows != 0 ? a.gate_rows : 1;
  size_t const runs = dlmi_ceil_div(B, gr);
  dlmi_span const spans[] = {{dx, B * row, true}, {du, B * row, true}, {dgate, runs * row, false}, {dw_post, H * 4, false},
                             {db_post, H * 4, false}, {dw_pre, H * 4, false}, {db_pre, H * 4, false}, {u, B * row, true},
                             {y, B * row, true}, {dy, B * row, true}, {dh, B * row, true}, {gate, runs * row, false},
                             {w_post, H * 4, false}, {b_post, H * 4, false}, {w_pre, H * 4, false}};
  DLMI_REQUIRE(ctx, !dlmi_spans_collide(spans, 7, 15), "an output overlaps another array");
  a.u = u;
  a.y = const_cast<void *>(y);
  a.gate = gate;
  a.w_post = w_post;
  a.b_post = b_post;
  a.w_pre = w_pre;
  a.dy = dy;
  a.dh = dh;
  a.dx = dx;
  a.du = du;
  a.dgate = dgate;
  float *const params[4] = {dw_post, db_post, dw_pre, db_pre};
  for (int k = 0; k < 4; ++k) a.plane[k] = params[k] != nullptr ? a.planes++ : -1;
  unsigned const sums = static_cast<unsigned>(a.planes);
  // as many workgroups as run at once (16 wavefronts per CU), but at least 4 rows each where there are sums: a workgroup
  // leaves a row of partial sums per plane
  size_t const nt = static_cast<size_t>(bn_threads(a.H, bn_each(type, true)));
  size_t const most = static_cast<size_t>(ctx->num_cu) * (nt < 1024 ? 1024 / nt : 1);
  size_t want = dlmi_ceil_div(B, most);
  if ((sums != 0 || gr > 1) && want < 4) want = 4;
  size_t blocks;
  a.slices = 1;
  a.direct = gr <= want ? 1 : 0;
  if (a.direct) {
    a.rows_per_wg = want / gr * gr;
    blocks = dlmi_ceil_div(B, a.rows_per_wg);
  } else {
    // (runs that are cut into slices are longer than `want` rows, so there are fewer of them than workgroups)
    a.slices = static_cast<unsigned>(dlmi_ceil_div(gr < B ? gr : B, want));
    a.rows_per_wg = want;
    blocks = runs * a.slices;
  }
  a.plane[4] = !a.direct && dgate != nullptr ? a.planes++ : -1;
  if (a.planes != 0) {
    int const rc = dlmi_scratch_reserve(ctx, blocks * a.planes * H * sizeof(float));
    if (rc != DLMI_OK) return rc;
    a.partial = reinterpret_cast<float *>(dlmi_scratch_data(ctx));
  }
  bn_dispatch(ctx, type, true, a, static_cast<unsigned>(blocks));
  DLMI_LAUNCH_CHECK(ctx, "k_block_norm_bwd");
  if (a.partial == nullptr) return DLMI_OK;
  // (without dh nothing was added up for the norm before the next block: the kernel left zeros)
  BnReduce r = {};
  r.partial = a.partial;
  for (int k = 0; k < 5; ++k) r.plane[k] = a.plane[k];
  for (int k = 0; k < 4; ++k) r.out[k] = params[k];
  r.planes = a.planes;
  r.dgate = dgate;
  r.workgroups = static_cast<unsigned>(blocks);
  r.slices = a.slices;
  r.H = a.H;
  r.accumulate = accumulate;
  dim3 const grid(static_cast<unsigned>(dlmi_ceil_div(H, 64)), sums + (a.plane[4] >= 0 ? static_cast<unsigned>(runs) : 0u));
  if (type == DLMI_F32)
    hipLaunchKernelGGL(k_block_norm_reduce<float>, grid, dim3(1024), 0, ctx->stream, r, sums);
  else
    hipLaunchKernelGGL(k_block_norm_reduce<__bf16>, grid, dim3(1024), 0, ctx->stream, r, sums);
  DLMI_LAUNCH_CHECK(ctx, "k_block_norm_reduce");
  return DLMI_OK;
}

}  // extern "C"
