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

template <class T>
constexpr int kBnVec = 16 / static_cast<int>(sizeof(T));  // elements of a 16-byte access

template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) BnVec {
  T v[kBnVec<T>];
};

// 16 bytes at a time whatever the alignment of the row (the hardware takes unaligned 16-byte accesses).
template <class T, int N>
__device__ __forceinline__ void bn_load(T const *row, int col, int H, float (&o)[N]) {
  if (col + N <= H) {
    BnVec<T> const v = *reinterpret_cast<BnVec<T> const *>(row + col);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = static_cast<float>(v.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = col + i < H ? static_cast<float>(row[col + i]) : 0.0f;
  }
}
template <class T, int N>
__device__ __forceinline__ void bn_store(T *row, int col, int H, float const (&o)[N]) {
  if (col + N <= H) {
    BnVec<T> v;
#pragma unroll
    for (int i = 0; i < N; ++i) v.v[i] = static_cast<T>(o[i]);
    *reinterpret_cast<BnVec<T> *>(row + col) = v;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (col + i < H) row[col + i] = static_cast<T>(o[i]);
  }
}
template <int N>
__device__ __forceinline__ void bn_param(float const *p, float dflt, int col, int H, float (&o)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = p != nullptr && col + i < H ? p[col + i] : dflt;
}

// Sums of two values over the NT threads of a row, the same in every thread.
template <int NT>
__device__ __forceinline__ void bn_sum2(float &a, float &b, float2 *lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    a += __shfl_xor(a, o);
    b += __shfl_xor(b, o);
  }
  if constexpr (NT > 64) {
    __syncthreads();  // the previous sums have been read
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = make_float2(a, b);
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
      a += lds[w].x;
      b += lds[w].y;
    }
  }
}

__device__ __forceinline__ float bn_gate(int act, float g) {
  if (act == DLMI_ACT_SIGMOID) return 1.0f / (1.0f + expf(-g));
  if (act == DLMI_ACT_TANH) return tanhf(g);
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
  float *partial;       // [workgroups][5][H]: dw_post, db_post, dw_pre, db_pre, the gate's
  int want_gate_direct;  // a workgroup covers whole runs of rows that share a gate: it writes dgate itself
  size_t B;
  int H;
  int post, pre, act;
  size_t gate_rows;     // 0: no gate
  size_t rows_per_wg;   // direct: rows of a workgroup (a multiple of gate_rows); otherwise rows of a slice
  unsigned slices;      // of a run of gate_rows rows
  float rs, bs, eps_post, eps_pre;
};

template <class T, int NT, int C>
__global__ __launch_bounds__(NT) void k_block_norm_fwd(BnArgs a) {
  constexpr int N = kBnVec<T>;
  __shared__ float2 lds[16];
  int const H = a.H;
  float const inv_h = 1.0f / static_cast<float>(H);
  float w1[C][N], b1[C][N], w2[C][N], b2[C][N];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    int const col = (c * NT + threadIdx.x) * N;
    bn_param(a.w_post, 1.0f, col, H, w1[c]);
    bn_param(a.b_post, 0.0f, col, H, b1[c]);
    bn_param(a.w_pre, 1.0f, col, H, w2[c]);
    bn_param(a.b_pre, 0.0f, col, H, b2[c]);
  }
  for (size_t r = blockIdx.x; r < a.B; r += gridDim.x) {
    size_t const at = r * static_cast<size_t>(H);
    float u[C][N], x[C][N], g[C][N];
#pragma unroll
    for (int c = 0; c < C; ++c) bn_load(static_cast<T const *>(a.u) + at, (c * NT + threadIdx.x) * N, H, u[c]);
#pragma unroll
    for (int c = 0; c < C; ++c) bn_load(static_cast<T const *>(a.x) + at, (c * NT + threadIdx.x) * N, H, x[c]);
    if (a.gate_rows != 0) {
      T const *const gr = static_cast<T const *>(a.gate) + (a.gate_rows == 1 ? r : r / a.gate_rows) * static_cast<size_t>(H);
#pragma unroll
      for (int c = 0; c < C; ++c) bn_load(gr, (c * NT + threadIdx.x) * N, H, g[c]);
    }
    // the columns beyond the row are zero in u and x; what centring makes of them stays out of the sums
    auto const norm = [&](float (&v)[C][N], int how, float eps) {
      if (how == DLMI_ROW_NORM_NONE) return;
      float s = 0.0f, q = 0.0f;
      if (how == DLMI_ROW_NORM_LAYER) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int i = 0; i < N; ++i) s += v[c][i];
        bn_sum2<NT>(s, q, lds);
        float const mean = s * inv_h;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int i = 0; i < N; ++i) v[c][i] = (c * NT + threadIdx.x) * N + i < static_cast<unsigned>(H) ? v[c][i] - mean : 0.0f;
        s = q = 0.0f;
      }
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < N; ++i) q += v[c][i] * v[c][i];
      bn_sum2<NT>(s, q, lds);
      float const rstd = 1.0f / sqrtf(q * inv_h + eps);
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < N; ++i) v[c][i] *= rstd;
    };
    norm(u, a.post, a.eps_post);
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float n = u[c][i] * w1[c][i] + b1[c][i];
        if (a.gate_rows != 0) n *= bn_gate(a.act, g[c][i]);
        x[c][i] = a.rs * x[c][i] + a.bs * n;
      }
      bn_store(static_cast<T *>(a.y) + at, (c * NT + threadIdx.x) * N, H, x[c]);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if ((c * NT + threadIdx.x) * N + i >= static_cast<unsigned>(H)) x[c][i] = 0.0f;
    }
    norm(x, a.pre, a.eps_pre);
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[c][i] = x[c][i] * w2[c][i] + b2[c][i];
      bn_store(static_cast<T *>(a.h) + at, (c * NT + threadIdx.x) * N, H, x[c]);
    }
  }
}

template <class T, int NT, int C>
__global__ __launch_bounds__(NT) void k_block_norm_bwd(BnArgs a) {
  constexpr int N = kBnVec<T>;
  __shared__ float2 lds[16];
  int const H = a.H;
  float const inv_h = 1.0f / static_cast<float>(H);
  float w1[C][N], b1[C][N], w2[C][N];
  float dw1[C][N], db1[C][N], dw2[C][N], db2[C][N], dg[C][N];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    int const col = (c * NT + threadIdx.x) * N;
    bn_param(a.w_post, 1.0f, col, H, w1[c]);
    bn_param(a.b_post, 0.0f, col, H, b1[c]);
    bn_param(a.w_pre, 1.0f, col, H, w2[c]);
#pragma unroll
    for (int i = 0; i < N; ++i) dw1[c][i] = db1[c][i] = dw2[c][i] = db2[c][i] = dg[c][i] = 0.0f;
  }
  size_t r0, r1;
  if (a.want_gate_direct) {
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
  for (size_t r = r0; r < r1; ++r) {
    size_t const at = r * static_cast<size_t>(H);
    float u[C][N], y[C][N], t[C][N], e[C][N], g[C][N];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      int const col = (c * NT + threadIdx.x) * N;
      bn_load(static_cast<T const *>(a.u) + at, col, H, u[c]);
      if (live_y) bn_load(static_cast<T const *>(a.y) + at, col, H, y[c]);
      if (a.dy != nullptr) {
        bn_load(static_cast<T const *>(a.dy) + at, col, H, t[c]);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) t[c][i] = 0.0f;
      }
      if (a.dh != nullptr) bn_load(static_cast<T const *>(a.dh) + at, col, H, e[c]);
    }
    if (a.gate_rows != 0) {
      T const *const gr = static_cast<T const *>(a.gate) + (a.gate_rows == 1 ? r : r / a.gate_rows) * static_cast<size_t>(H);
#pragma unroll
      for (int c = 0; c < C; ++c) bn_load(gr, (c * NT + threadIdx.x) * N, H, g[c]);
    }
    // the means, where a layer norm asks for them
    if (a.post == DLMI_ROW_NORM_LAYER || (live_y && a.pre == DLMI_ROW_NORM_LAYER)) {
      float su = 0.0f, sy = 0.0f;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          su += u[c][i];
          if (live_y) sy += y[c][i];
        }
      bn_sum2<NT>(su, sy, lds);
      float const mu = a.post == DLMI_ROW_NORM_LAYER ? su * inv_h : 0.0f;
      float const my = a.pre == DLMI_ROW_NORM_LAYER ? sy * inv_h : 0.0f;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          bool const in = (c * NT + threadIdx.x) * N + i < static_cast<unsigned>(H);
          u[c][i] = in ? u[c][i] - mu : 0.0f;
          if (live_y) y[c][i] = in ? y[c][i] - my : 0.0f;
        }
    }
    // pre's gradient
    float qu = 0.0f, qy = 0.0f, sg = 0.0f, sgy = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        qu += u[c][i] * u[c][i];
        if (live_y) {
          float const gh = e[c][i] * w2[c][i];
          qy += y[c][i] * y[c][i];
          sg += gh;
          sgy += gh * y[c][i];
        }
      }
    bn_sum2<NT>(qu, qy, lds);
    float const ru = a.post != DLMI_ROW_NORM_NONE ? 1.0f / sqrtf(qu * inv_h + a.eps_post) : 1.0f;
    if (live_y) {
      bn_sum2<NT>(sg, sgy, lds);
      float const ry = 1.0f / sqrtf(qy * inv_h + a.eps_pre);
      float const c1 = a.pre == DLMI_ROW_NORM_LAYER ? sg * inv_h : 0.0f;
      float const c2 = sgy * ry * inv_h;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          float const yh = y[c][i] * ry;
          dw2[c][i] += e[c][i] * yh;
          db2[c][i] += e[c][i];
          t[c][i] += ry * (e[c][i] * w2[c][i] - c1 - yh * c2);
        }
    } else if (a.dh != nullptr) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < N; ++i) t[c][i] += e[c][i];
    }
    // the gate, then post's gradient; e becomes dn, y becomes dx
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        bool const in = (c * NT + threadIdx.x) * N + i < static_cast<unsigned>(H);
        float const uh = u[c][i] * ru;
        float d = a.bs * t[c][i];
        if (a.gate_rows != 0) {
          float const f = bn_gate(a.act, g[c][i]);
          dg[c][i] += d * bn_gate_slope(a.act, f) * (uh * w1[c][i] + b1[c][i]);
          d *= f;
        }
        d = in ? d : 0.0f;
        dw1[c][i] += d * uh;
        db1[c][i] += d;
        float const gd = d * w1[c][i];
        s1 += gd;
        s2 += gd * uh;
        e[c][i] = d;
        t[c][i] *= a.rs;
        u[c][i] = uh;
      }
      bn_store(static_cast<T *>(a.dx) + at, (c * NT + threadIdx.x) * N, H, t[c]);
    }
    if (a.post != DLMI_ROW_NORM_NONE) {
      bn_sum2<NT>(s1, s2, lds);
      float const c1 = a.post == DLMI_ROW_NORM_LAYER ? s1 * inv_h : 0.0f, c2 = s2 * inv_h;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < N; ++i) e[c][i] = ru * (e[c][i] * w1[c][i] - c1 - u[c][i] * c2);
    }
#pragma unroll
    for (int c = 0; c < C; ++c) bn_store(static_cast<T *>(a.du) + at, (c * NT + threadIdx.x) * N, H, e[c]);
    if (a.want_gate_direct && a.gate_rows != 0 && ((r + 1) % a.gate_rows == 0 || r + 1 == a.B)) {
      T *const out = static_cast<T *>(a.dgate) + r / a.gate_rows * static_cast<size_t>(H);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if (a.dgate != nullptr) bn_store(out, (c * NT + threadIdx.x) * N, H, dg[c]);
#pragma unroll
        for (int i = 0; i < N; ++i) dg[c][i] = 0.0f;
      }
    }
  }
  if (a.partial == nullptr) return;
  float *const out = a.partial + static_cast<size_t>(blockIdx.x) * 5 * H;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      int const col = (c * NT + threadIdx.x) * N + i;
      if (col >= H) continue;
      if (a.post != DLMI_ROW_NORM_NONE) {
        out[col] = dw1[c][i];
        out[H + col] = db1[c][i];
      }
      if (a.pre != DLMI_ROW_NORM_NONE) {
        out[2 * H + col] = dw2[c][i];
        out[3 * static_cast<size_t>(H) + col] = db2[c][i];
      }
      if (!a.want_gate_direct) out[4 * static_cast<size_t>(H) + col] = dg[c][i];
    }
}

struct BnReduce {
  float const *partial;
  float *out[4];      // the parameters' gradients (may be null)
  void *dgate;        // [runs][H] (may be null)
  unsigned workgroups, slices, runs;
  int H, accumulate;
};

// 64 columns of one plane: 16 threads per column add every 16th row, then a tree.  Planes 0-3 the parameters' gradients
// over all workgroups, planes 4 and up a run's slices of the gate's.
template <class T>
__global__ __launch_bounds__(1024) void k_block_norm_reduce(BnReduce a) {
  __shared__ float lds[16][64];
  unsigned const plane = blockIdx.y < 4 ? blockIdx.y : 4;
  if (plane < 4 ? a.out[plane] == nullptr : a.dgate == nullptr) return;
  unsigned const from = plane < 4 ? 0 : (blockIdx.y - 4) * a.slices, n = plane < 4 ? a.workgroups : a.slices;
  int const col = static_cast<int>(blockIdx.x * 64 + (threadIdx.x & 63));
  unsigned const part = threadIdx.x >> 6;
  float s = 0.0f;
  if (col < a.H)
    for (unsigned w = part; w < n; w += 16) s += a.partial[(static_cast<size_t>(from + w) * 5 + plane) * a.H + col];
  lds[part][threadIdx.x & 63] = s;
  __syncthreads();
  for (unsigned o = 8; o > 0; o >>= 1) {
    if (part < o) lds[part][threadIdx.x & 63] += lds[part + o][threadIdx.x & 63];
    __syncthreads();
  }
  if (part != 0 || col >= a.H) return;
  s = lds[0][threadIdx.x & 63];
  if (plane < 4)
    a.out[plane][col] = a.accumulate ? a.out[plane][col] + s : s;
  else
    static_cast<T *>(a.dgate)[static_cast<size_t>(blockIdx.y - 4) * a.H + col] = static_cast<T>(s);
}

template <class T, int NT, int C>
static void bn_launch(dlmi_ctx *ctx, bool back, BnArgs const &a, unsigned blocks) {
  if (back)
    hipLaunchKernelGGL((k_block_norm_bwd<T, NT, C>), dim3(blocks), dim3(NT), 0, ctx->stream, a);
  else
    hipLaunchKernelGGL((k_block_norm_fwd<T, NT, C>), dim3(blocks), dim3(NT), 0, ctx->stream, a);
}

// Threads of a row: 8 columns each, up to 1024 threads; wider rows 16 columns each.
static int bn_threads(int H) {
  int nt = 64;
  while (nt < 1024 && nt * 8 < H) nt *= 2;
  return nt;
}

template <class T>
static void bn_dispatch(dlmi_ctx *ctx, bool back, BnArgs const &a, unsigned blocks) {
  constexpr int C = 8 / kBnVec<T>;
  switch (bn_threads(a.H)) {
    case 64: return bn_launch<T, 64, C>(ctx, back, a, blocks);
    case 128: return bn_launch<T, 128, C>(ctx, back, a, blocks);
    case 256: return bn_launch<T, 256, C>(ctx, back, a, blocks);
    case 512: return bn_launch<T, 512, C>(ctx, back, a, blocks);
    default:
      if (a.H <= 8192) return bn_launch<T, 1024, C>(ctx, back, a, blocks);
      return bn_launch<T, 1024, 2 * C>(ctx, back, a, blocks);
  }
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
  a.gate_rows = d->gate_rows;
  a.rs = d->residual_scale;
  a.bs = d->branch_scale;
  a.eps_post = d->eps_post;
  a.eps_pre = d->eps_pre;
  return a;
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
  BnArgs a = bn_args(desc, B, H);
  a.x = x;
  a.u = u;
  a.gate = gate;
  a.w_post = w_post;
  a.b_post = b_post;
  a.w_pre = w_pre;
  a.b_pre = b_pre;
  a.y = y;
  a.h = h;
  size_t blocks = static_cast<size_t>(ctx->num_cu) * (2048 / bn_threads(a.H));
  if (blocks > B) blocks = B;
  if (type == DLMI_F32)
    bn_dispatch<float>(ctx, false, a, static_cast<unsigned>(blocks));
  else
    bn_dispatch<__bf16>(ctx, false, a, static_cast<unsigned>(blocks));
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
  if (B * H == 0) return DLMI_OK;
  DLMI_REQUIRE_DEVICE(ctx);
  DLMI_REQUIRE(ctx, u != nullptr && dx != nullptr && du != nullptr, "null pointer");
  DLMI_REQUIRE(ctx, dy != nullptr || dh != nullptr, "no gradient to start from");
  DLMI_REQUIRE(ctx, y != nullptr || dh == nullptr || desc->pre == DLMI_ROW_NORM_NONE, "null pointer");
  BnArgs a = bn_args(desc, B, H);
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
  bool const sums = dw_post != nullptr || db_post != nullptr || dw_pre != nullptr || db_pre != nullptr;
  // as many workgroups as fill the device with 32 wavefronts per CU, but at least 4 rows each where there are sums: a
  // workgroup leaves up to 5 rows of partial sums
  size_t most = static_cast<size_t>(ctx->num_cu) * (2048 / bn_threads(a.H));
  size_t want = dlmi_ceil_div(B, most);
  if ((sums || desc->gate_rows > 1) && want < 4) want = 4;
  size_t const gr = desc->gate_rows != 0 ? desc->gate_rows : 1;
  size_t runs = dlmi_ceil_div(B, gr), blocks;
  a.slices = 1;
  a.want_gate_direct = gr <= want ? 1 : 0;
  if (a.want_gate_direct) {
    a.rows_per_wg = want / gr * gr;
    blocks = dlmi_ceil_div(B, a.rows_per_wg);
  } else {
    a.slices = static_cast<unsigned>(dlmi_ceil_div(gr < B ? gr : B, want));
    a.rows_per_wg = want;
    blocks = runs * a.slices;
  }
  // (runs that are cut into slices are longer than `want` rows, so there are fewer of them than workgroups)
  if (sums || (!a.want_gate_direct && dgate != nullptr)) {
    int const rc = dlmi_scratch_reserve(ctx, blocks * 5 * H * sizeof(float));
    if (rc != DLMI_OK) return rc;
    a.partial = reinterpret_cast<float *>(dlmi_scratch_data(ctx));
  }
  if (type == DLMI_F32)
    bn_dispatch<float>(ctx, true, a, static_cast<unsigned>(blocks));
  else
    bn_dispatch<__bf16>(ctx, true, a, static_cast<unsigned>(blocks));
  DLMI_LAUNCH_CHECK(ctx, "k_block_norm_bwd");
  if (a.partial == nullptr) return DLMI_OK;
  BnReduce r = {};
  r.partial = a.partial;
  r.out[0] = dw_post;
  r.out[1] = db_post;
  // without dh nothing was added up for the norm before the next block: the kernel left zeros
  r.out[2] = dw_pre;
  r.out[3] = db_pre;
  r.dgate = a.want_gate_direct ? nullptr : dgate;
  r.workgroups = static_cast<unsigned>(blocks);
  r.slices = a.slices;
  r.runs = static_cast<unsigned>(runs);
  r.H = a.H;
  r.accumulate = accumulate;
  dim3 const grid(static_cast<unsigned>(dlmi_ceil_div(H, 64)), 4 + (r.dgate != nullptr ? r.runs : 0));
  if (type == DLMI_F32)
    hipLaunchKernelGGL(k_block_norm_reduce<float>, grid, dim3(1024), 0, ctx->stream, r);
  else
    hipLaunchKernelGGL(k_block_norm_reduce<__bf16>, grid, dim3(1024), 0, ctx->stream, r);
  DLMI_LAUNCH_CHECK(ctx, "k_block_norm_reduce");
  return DLMI_OK;
}

}  // extern "C"
