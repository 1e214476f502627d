// Matrix products on the 16-bit matrix pipe: the K loop that the Muon step (muon_kernels.hip) and the vocabulary cross
// entropy (vocab_ce.hip) share, and the operand format it reads.
//
// C[i][j] = sum_k P[i][k] Q[j][k], both operands given as "packed" matrices: 32 rows x 16 k are one fragment of
// 1 KiB, lane l of a wavefront holding row l & 31 and the 8 consecutive k from 8 (l >> 5), which is how
// v_mfma_f32_32x32x16_f16 takes its operands.  Fragments lie [row block][k block][plane].  So a fragment goes from
// memory to LDS as one 16-byte-per-lane direct load, is read back as one ds_read_b128 in lane order (no bank is hit
// twice), and the loop has no bounds to check: whoever packs pads rows and k with zeros.
//
// Planes.  One plane holds a value rounded to f16 (11 significant bits: what a bf16 input has, and more).  Two planes
// hold x = hi + lo, each f16, 22 bits in all; the product is hi hi + hi lo + lo hi, three matrix instructions, accumulated
// in fp32.  The dropped lo lo is below 2^-22 of a term, so the result is as good as a product of fp32 values, at a third
// of the 16-bit rate = 833 TFLOP/s against 157 TFLOP/s on the fp32 matrix pipe.  f16 has 5 exponent bits: the packer
// multiplies by a power of two so that the largest magnitude lies near the top of the range; what is 2^-18 of it or
// smaller loses bits of its lo (an absolute error below 2^-40 of the largest).
#pragma once

#include "dlmi_common.hpp"

namespace dlmi {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kFragBytes = 1024;

// Bytes of a packed matrix of `rows` x `k` (both already padded: rows to 32, k to 16).
inline size_t packed_bytes(size_t rows, size_t k, int planes) { return rows * k * 2 * planes; }

// Workgroup number -> number in an order in which the workgroups of one XCD (numbers equal modulo 8) are consecutive.
__device__ __forceinline__ unsigned xcd_consecutive(unsigned id, unsigned n) {
  unsigned const q = n >> 3, r = n & 7, x = id & 7;
  return x * q + (x < r ? x : r) + (id >> 3);
}

// One step of the K loop reads one stage of LDS: KS k blocks of all planes of the BM + BN rows, four stages in all.  64 x 64
// tiles take twice the k blocks of the others per stage: their stages are short, and three of them ahead is less than a load
// takes.
template <int BM, int BN, int NP>
struct HalfTile {
  static constexpr int kPlanes = NP;
  static constexpr int kDepth = BM + BN <= 128 ? 4 : 2;      // fragments of a row block in a stage
  static constexpr int KS = kDepth / NP;                     // k blocks per stage
  static constexpr int kMB = BM / 64, kNB = BN / 64;         // 32 x 32 blocks of a wavefront, 2 x 2 wavefronts
  static constexpr int kFragsA = BM / 32 * kDepth, kFragsB = BN / 32 * kDepth;  // fragments of a stage
  static constexpr int kStageBytes = (kFragsA + kFragsB) * kFragBytes;
  static constexpr int kLoads = (kFragsA + kFragsB) / 4;     // direct loads of a wavefront per stage
  static constexpr int kStep = KS * NP * kFragBytes;         // bytes from a row block's stage to its next
  // where fragment f of an operand's stage lies in its row block: plane f % NP of k block f / NP
  static __host__ __device__ constexpr int at(int f) { return f % kDepth * kFragBytes; }
};

template <class T>
struct HalfAcc {
  f32x16 v[T::kMB][T::kNB];
};

template <class T>
__device__ __forceinline__ void half_stage_load(char *lds, char const *P, char const *Q, size_t row_stride_p,
                                                size_t row_stride_q, int wave, int lane) {
  // fragment f of an operand: of row block f / kDepth
#pragma unroll
  for (int u = 0; u < T::kFragsA / 4; ++u) {
    int const f = u * 4 + wave;
    char const *src = P + static_cast<size_t>(f / T::kDepth) * row_stride_p + T::at(f) + lane * 16;
    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void const *)src,
                                     (__attribute__((address_space(3))) void *)(lds + f * kFragBytes), 16, 0, 0);
  }
#pragma unroll
  for (int u = 0; u < T::kFragsB / 4; ++u) {
    int const f = u * 4 + wave;
    char const *src = Q + static_cast<size_t>(f / T::kDepth) * row_stride_q + T::at(f) + lane * 16;
    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void const *)src,
                                     (__attribute__((address_space(3))) void *)(lds + (T::kFragsA + f) * kFragBytes), 16,
                                     0, 0);
  }
}

// The fragments of one k block (all planes) that a wavefront multiplies.
template <class T>
struct HalfFrags {
  half8 p[T::kPlanes][T::kMB], q[T::kPlanes][T::kNB];
};

template <class T>
__device__ __forceinline__ void half_frags_read(HalfFrags<T> &f, char const *lds, int ks, int wm, int wn, int lane) {
#pragma unroll
  for (int pl = 0; pl < T::kPlanes; ++pl) {
#pragma unroll
    for (int m = 0; m < T::kMB; ++m)
      f.p[pl][m] = *reinterpret_cast<half8 const *>(lds + (((wm * T::kMB + m) * T::kDepth + ks * T::kPlanes + pl) * kFragBytes + lane * 16));
#pragma unroll
    for (int n = 0; n < T::kNB; ++n)
      f.q[pl][n] = *reinterpret_cast<half8 const *>(
          lds + ((T::kFragsA + (wn * T::kNB + n) * T::kDepth + ks * T::kPlanes + pl) * kFragBytes + lane * 16));
  }
}

template <class T>
__device__ __forceinline__ void half_mfma(HalfAcc<T> &acc, HalfFrags<T> const &f) {
#pragma unroll
  for (int t = 0; t < (T::kPlanes == 2 ? 3 : 1); ++t) {
    int const pp = t == 2 ? 1 : 0, qp = t == 1 ? 1 : 0;
#pragma unroll
    for (int m = 0; m < T::kMB; ++m)
#pragma unroll
      for (int n = 0; n < T::kNB; ++n)
        acc.v[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.p[pp][m], f.q[qp][n], acc.v[m][n], 0, 0, 0);
  }
}

// Waits until at most the last `flying` stages requested are still on their way and this wavefront's own LDS reads are
// done, then lets all wavefronts of the workgroup pass together.  (The empty asm statements keep the compiler from
// moving LDS accesses across the barrier, which by itself is no fence.)
template <class T, int flying>
__device__ __forceinline__ void half_stage_wait() {
  constexpr int n = flying * T::kLoads;
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (n & 15) | ((n >> 4) << 14));  // vmcnt(n) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The order of a k block's instructions: the next block's LDS reads and the next stages' loads spread between the matrix
// instructions.  Left to itself the compiler puts them behind most of these, and the loads right before the next wait: 246
// us against 221 us for 8192 x 8192 x 2048 in one plane (1242 TFLOP/s by itself; 1150 - 1270 in the kernels that use it), 623
// against 603 us in two (1368 TFLOP/s), 50 against 45 us for 2048^3 in two planes with 128 x 128 tiles.  One plane of a 256 x
// 256 tile has few matrix instructions per read and does best with all reads first (221 against 224 us); everything else with
// reads and loads spread alike.
template <class T, bool LOADS>
__device__ __forceinline__ void half_schedule() {
  constexpr int kMfma = 0x008, kLoad = 0x020, kRead = 0x100;
  constexpr int NM = T::kMB * T::kNB * (T::kPlanes == 2 ? 3 : 1), NR = (T::kMB + T::kNB) * T::kPlanes;
  if constexpr (T::kPlanes == 1 && T::kMB == 4) {
    __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      __builtin_amdgcn_sched_group_barrier(kRead, 1, 0);
      __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
    }
    if constexpr (LOADS) {
#pragma unroll
      for (int i = 0; i < T::kLoads; ++i) {
        __builtin_amdgcn_sched_group_barrier(kLoad, 1, 0);
        __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      if (LOADS && i < T::kLoads) __builtin_amdgcn_sched_group_barrier(kLoad, 1, 0);
      __builtin_amdgcn_sched_group_barrier(kRead, 1, 0);
      __builtin_amdgcn_sched_group_barrier(kMfma, NM / NR, 0);
    }
  }
}

// 64 x 64 tiles: a wavefront has one block, so a k block is three matrix instructions at most, less than an LDS read takes.  The
// fragments of a whole stage are read while those of the one before are multiplied; who passes the barrier has all of its
// stage in registers, so the buffer is filled again at once, and up to four stages are on their way.  Loads are made without
// conditions, beyond the end of the last stage again (of any other order the compiler knows too little, and waits for all
// loads before it reads LDS).
template <class T>
__device__ __forceinline__ void half_gemm_short(HalfAcc<T> &acc, char *buf0, char *buf1, char *buf2, char *buf3, char const *P, char const *Q,
                                                size_t row_stride_p, size_t row_stride_q, int stages, int wm, int wn, int wave, int lane) {
  char *const bufs[4] = {buf0, buf1, buf2, buf3};
  auto const load = [&](char *buf, int t) {
    t = t < stages ? t : stages - 1;
    half_stage_load<T>(buf, P + static_cast<size_t>(t) * T::kStep, Q + static_cast<size_t>(t) * T::kStep, row_stride_p, row_stride_q, wave, lane);
  };
  HalfFrags<T> cur[T::KS], nxt[T::KS];
#pragma unroll
  for (int u = 0; u < 4; ++u) load(bufs[u], u);
  half_stage_wait<T, 3>();
#pragma unroll
  for (int ks = 0; ks < T::KS; ++ks) half_frags_read<T>(cur[ks], bufs[0], ks, wm, wn, lane);
  auto const step = [&](char *free, char const *next, int t) {
    half_stage_wait<T, 2>();
    load(free, t + 4);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int ks = 0; ks < T::KS; ++ks) half_frags_read<T>(nxt[ks], next, ks, wm, wn, lane);
#pragma unroll
    for (int ks = 0; ks < T::KS; ++ks) half_mfma<T>(acc, cur[ks]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // (8 reads, 4 or 6 matrix instructions)
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int ks = 0; ks < T::KS; ++ks) cur[ks] = nxt[ks];
  };
  int t = 0;
  for (; t + 4 <= stages; t += 4) {
    step(buf0, buf1, t);
    step(buf1, buf2, t + 1);
    step(buf2, buf3, t + 2);
    step(buf3, buf0, t + 3);
  }
  if (t < stages) {
    step(buf0, buf1, t);
    if (t + 1 < stages) {
      step(buf1, buf2, t + 1);
      if (t + 2 < stages) step(buf2, buf3, t + 2);
    }
  }
  half_stage_wait<T, 0>();  // nothing may land in LDS that is no longer this workgroup's
}

// The K loop of one workgroup (256 threads, wavefronts 2 x 2) over `stages` >= 1 stages.  P, Q: the first fragment of the
// tile's first row block at the first k block; row_stride_*: bytes from one row block to the next.
template <class T>
__device__ __forceinline__ void half_gemm(HalfAcc<T> &acc, char const *P, char const *Q, size_t row_stride_p, size_t row_stride_q, int stages) {
  __shared__ __attribute__((aligned(1024))) char buf0[T::kStageBytes];
  __shared__ __attribute__((aligned(1024))) char buf1[T::kStageBytes];
  __shared__ __attribute__((aligned(1024))) char buf2[T::kStageBytes];
  __shared__ __attribute__((aligned(1024))) char buf3[T::kStageBytes];
  char *const bufs[4] = {buf0, buf1, buf2, buf3};
  int const lane = threadIdx.x & 63;
  int const wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int const wm = wave >> 1, wn = wave & 1;
#pragma unroll
  for (int m = 0; m < T::kMB; ++m)
#pragma unroll
    for (int n = 0; n < T::kNB; ++n) acc.v[m][n] = f32x16{};
  if constexpr (T::kMB == 1) {
    half_gemm_short<T>(acc, buf0, buf1, buf2, buf3, P, Q, row_stride_p, row_stride_q, stages, wm, wn, wave, lane);
    return;
  }

  auto const load = [&](char *buf, int t) {
    half_stage_load<T>(buf, P + static_cast<size_t>(t) * T::kStep, Q + static_cast<size_t>(t) * T::kStep, row_stride_p, row_stride_q, wave, lane);
  };
  // the first three stages are requested before the first is waited for
  load(bufs[0], 0);
  if (stages > 1) load(bufs[1], 1);
  if (stages > 2) load(bufs[2], 2);
  if (stages > 2)
    half_stage_wait<T, 2>();
  else if (stages > 1)
    half_stage_wait<T, 1>();
  else
    half_stage_wait<T, 0>();
  HalfFrags<T> cur, nxt;
  half_frags_read<T>(cur, bufs[0], 0, wm, wn, lane);
  // One stage: the fragments of a k block are multiplied while those of the next are read.  Before the last k block is
  // multiplied the next stage has landed and every wavefront has read all of the stage before this one, whose buffer
  // is then filled again.
  int t0 = 0;
  for (; t0 + 6 < stages; t0 += 4) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int ks = 0; ks < T::KS; ++ks) {
        __builtin_amdgcn_sched_barrier(0);
        if (ks + 1 < T::KS) {
          half_frags_read<T>(nxt, bufs[u], ks + 1, wm, wn, lane);
        } else {
          half_stage_wait<T, 1>();
          load(bufs[(u + 3) & 3], t0 + u + 3);
          half_frags_read<T>(nxt, bufs[(u + 1) & 3], 0, wm, wn, lane);
        }
        half_mfma<T>(acc, cur);
        cur = nxt;
        if (ks + 1 == T::KS)
          half_schedule<T, true>();
        else
          half_schedule<T, false>();
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  for (; t0 < stages; t0 += 4) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      int const t = t0 + u;
      if (t < stages) {
#pragma unroll
        for (int ks = 0; ks < T::KS; ++ks) {
          if (ks + 1 < T::KS) {
            half_frags_read<T>(nxt, bufs[u], ks + 1, wm, wn, lane);
          } else if (t + 1 < stages) {
            if (t + 2 < stages)
              half_stage_wait<T, 1>();
            else
              half_stage_wait<T, 0>();
            if (t + 3 < stages) load(bufs[(u + 3) & 3], t + 3);
            half_frags_read<T>(nxt, bufs[(u + 1) & 3], 0, wm, wn, lane);
          }
          half_mfma<T>(acc, cur);
          cur = nxt;
        }
      }
    }
  }
}

// ---- the last tiles shared out -------------------------------------------------------------------------------------
// Of a number of tiles that is no multiple of the G workgroups that run at once, the last ones (fewer than G) would leave
// most of the device idle.  Their K loops are one list of pieces, kShareStages stages each, cut into G equal ranges; a
// workgroup leaves the sums of each part of a tile in its range in memory, and a second launch adds a tile's parts in the
// order of k and runs its epilogue, a wavefront per 32 x 32 block.
constexpr unsigned kShareStages = 4;

struct HalfShares {
  unsigned whole, tiles;    // tiles that have a workgroup each; all tiles
  unsigned stages;          // of a tile
  unsigned grid;            // workgroups of the shared tiles: every one of them has a piece
  unsigned pieces;          // of a shared tile
  unsigned long long total; // pieces of all shared tiles
  float *parts;             // [grid][2][BM * BN]: the first tile of a range, and the last
  // the workgroup that holds a piece, and the tile of a workgroup's first piece
  __host__ __device__ unsigned owner(unsigned long long piece) const { return static_cast<unsigned>(((piece + 1) * grid - 1) / total); }
  __host__ __device__ unsigned first(unsigned w) const { return static_cast<unsigned>(w * total / grid / pieces); }
};

// (Fewer shared tiles than workgroups: a range is shorter than a tile and touches at most two.)
inline HalfShares half_shares(unsigned tiles, unsigned stages, unsigned G, float *parts) {
  HalfShares s = {};
  s.tiles = tiles;
  s.whole = tiles - tiles % G;
  s.stages = stages;
  s.pieces = (stages + kShareStages - 1) / kShareStages;
  s.total = static_cast<unsigned long long>(tiles - s.whole) * s.pieces;
  s.grid = s.total < G ? static_cast<unsigned>(s.total) : G;
  s.parts = parts;
  return s;
}

// A wavefront's blocks of a part, register pairs of a block's 64 lanes side by side.
template <class T>
__device__ __forceinline__ void half_part_store(float *part, HalfAcc<T> const &acc) {
  f32x4 *const p = reinterpret_cast<f32x4 *>(part) + (threadIdx.x >> 6) * (T::kMB * T::kNB * 4 * 64) + (threadIdx.x & 63);
#pragma unroll
  for (int m = 0; m < T::kMB; ++m)
#pragma unroll
    for (int n = 0; n < T::kNB; ++n)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f32x16 const &v = acc.v[m][n];
        p[((m * T::kNB + n) * 4 + q) * 64] = f32x4{v[q * 4], v[q * 4 + 1], v[q * 4 + 2], v[q * 4 + 3]};
      }
}

// The parts of the shared tiles.  operands(tile, P, Q): a tile's operands at its first stage.
template <class T, class Operands>
__device__ __forceinline__ void half_gemm_parts(HalfShares const &s, size_t row_stride_p, size_t row_stride_q, Operands &&operands) {
  constexpr int kTile = 4 * T::kMB * T::kNB * 1024;
  unsigned const g = xcd_consecutive(blockIdx.x, gridDim.x);
  unsigned long long u = g * s.total / s.grid;
  unsigned long long const u1 = (g + 1ull) * s.total / s.grid;
  unsigned const first = static_cast<unsigned>(u / s.pieces);
  while (u < u1) {
    unsigned const shared = static_cast<unsigned>(u / s.pieces);
    unsigned long long const begin = static_cast<unsigned long long>(shared) * s.pieces, end = begin + s.pieces < u1 ? begin + s.pieces : u1;
    unsigned const from = static_cast<unsigned>(u - begin) * kShareStages, to = static_cast<unsigned>(end - begin) * kShareStages;
    char const *P, *Q;
    operands(s.whole + shared, P, Q);
    HalfAcc<T> acc;
    __syncthreads();  // the stages of the part before have been read
    half_gemm<T>(acc, P + static_cast<size_t>(from) * T::kStep, Q + static_cast<size_t>(from) * T::kStep, row_stride_p, row_stride_q,
                 static_cast<int>((to < s.stages ? to : s.stages) - from));
    half_part_store(s.parts + (static_cast<size_t>(g) * 2 + (shared == first ? 0 : 1)) * kTile, acc);
    u = end;
  }
}

// Block `block` (wavefront, m, n) of shared tile `shared`, its parts added in the order of k.
template <class T>
__device__ __forceinline__ f32x16 half_part_sum(HalfShares const &s, unsigned shared, unsigned block, int tile_floats) {
  unsigned long long const begin = static_cast<unsigned long long>(shared) * s.pieces;
  unsigned const w0 = s.owner(begin), w1 = s.owner(begin + s.pieces - 1);
  f32x16 v = {};
  for (unsigned w = w0; w <= w1; ++w) {
    float const *const part = s.parts + (static_cast<size_t>(w) * 2 + (shared == s.first(w) ? 0 : 1)) * tile_floats;
    f32x4 const *const p = reinterpret_cast<f32x4 const *>(part) + block * (4 * 64) + (threadIdx.x & 63);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      f32x4 const x = p[q * 64];
#pragma unroll
      for (int t = 0; t < 4; ++t) v[q * 4 + t] += x[t];
    }
  }
  return v;
}

// ---- a 32 x 32 block of C in registers (lane l: column j = l & 31, rows i = 8 (r >> 2) + 4 (l >> 5) + (r & 3)) -------------

// The block as two packed fragments of the transposed matrix (row j, k = i): k block 0 and 1.
struct HalfPair {
  half8 k0, k1;
};

__device__ __forceinline__ half8 half_join(half4 a, half4 b) {
  // rows 0-31 of a lane pair hold k 0-3 | 4-7 of two k octets: swapping the upper half of the first with the lower half
  // of the second leaves every lane one whole octet
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  u2 const ua = __builtin_bit_cast(u2, a), ub = __builtin_bit_cast(u2, b);
  auto const x = __builtin_amdgcn_permlane32_swap(ua[0], ub[0], false, false);
  auto const y = __builtin_amdgcn_permlane32_swap(ua[1], ub[1], false, false);
  u32x4 const r = {x[0], y[0], x[1], y[1]};
  return __builtin_bit_cast(half8, r);
}
__device__ __forceinline__ void half_part(half8 v, half4 &a, half4 &b) {  // the inverse
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  u32x4 const r = __builtin_bit_cast(u32x4, v);
  auto const x = __builtin_amdgcn_permlane32_swap(r[0], r[2], false, false);
  auto const y = __builtin_amdgcn_permlane32_swap(r[1], r[3], false, false);
  u2 const ua = {x[0], y[0]}, ub = {x[1], y[1]};
  a = __builtin_bit_cast(half4, ua);
  b = __builtin_bit_cast(half4, ub);
}

template <int NP>
struct HalfBlock {
  HalfPair pl[NP];
};

// Rounds the block to its planes (each to nearest even; the second holds what the first lost).  The empty asm makes the
// value one of fp32 before it is rounded: the compiler may otherwise fold a product before it into one of the two uses of
// `hi` (a multiplication that rounds to f16 at once), and a value near a tie then loses a whole step of its first plane.
template <int NP>
struct HalfQuads {
  half4 h[NP][4];  // [plane][r >> 2][r & 3]
};
template <int NP>
__device__ __forceinline__ HalfQuads<NP> half_planes(f32x16 const &v) {
  HalfQuads<NP> o;
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      float x = v[q * 4 + t];
      if constexpr (NP == 2) asm("" : "+v"(x));
      _Float16 const hi = static_cast<_Float16>(x);
      o.h[0][q][t] = hi;
      if constexpr (NP == 2) o.h[1][q][t] = static_cast<_Float16>(x - static_cast<float>(hi));
    }
  return o;
}
template <int NP>
__device__ __forceinline__ HalfBlock<NP> half_joined(HalfQuads<NP> const &q) {
  HalfBlock<NP> b;
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    b.pl[p].k0 = half_join(q.h[p][0], q.h[p][1]);
    b.pl[p].k1 = half_join(q.h[p][2], q.h[p][3]);
  }
  return b;
}
template <int NP>
__device__ __forceinline__ HalfBlock<NP> half_split(f32x16 const &v) {
  return half_joined<NP>(half_planes<NP>(v));
}

// dst: fragment (row block of j, k block of i) of the packed matrix; the block's second k block follows its planes.
template <int NP>
__device__ __forceinline__ void half_store(char *dst, HalfBlock<NP> const &b, int lane) {
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    *reinterpret_cast<half8 *>(dst + p * kFragBytes + lane * 16) = b.pl[p].k0;
    *reinterpret_cast<half8 *>(dst + (NP + p) * kFragBytes + lane * 16) = b.pl[p].k1;
  }
}

template <int NP>
__device__ __forceinline__ f32x16 half_load(char const *src, int lane) {
  f32x16 v = {};
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    half4 a[4];
    half_part(*reinterpret_cast<half8 const *>(src + p * kFragBytes + lane * 16), a[0], a[1]);
    half_part(*reinterpret_cast<half8 const *>(src + (NP + p) * kFragBytes + lane * 16), a[2], a[3]);
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int t = 0; t < 4; ++t) v[q * 4 + t] += static_cast<float>(a[q][t]);
  }
  return v;
}

// Lane l's octet of rows 0-15 (half 0) or 16-31 (half 1) of the 32-column identity.
__device__ __forceinline__ half8 half_identity(int half, int lane) {
  half8 r;
#pragma unroll
  for (int t = 0; t < 8; ++t) r[t] = static_cast<_Float16>((lane & 31) == half * 16 + (lane >> 5) * 8 + t ? 1.0f : 0.0f);
  return r;
}

// The plane of a block (fragments of the transposed matrix) times the identity: lane l then holds, in the layout of C, the
// transposed block (column i = l & 31, rows j).  One term per sum: exact.
__device__ __forceinline__ f32x16 half_transposed(HalfPair const &p, half8 id0, half8 id1) {
  f32x16 z = {};
  z = __builtin_amdgcn_mfma_f32_32x32x16_f16(p.k0, id0, z, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(p.k1, id1, z, 0, 0, 0);
}

// The same block packed the other way round (row i, k = j).
template <int NP>
__device__ __forceinline__ HalfBlock<NP> half_flip(HalfBlock<NP> const &b, half8 id0, half8 id1) {
  HalfBlock<NP> r;
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    f32x16 const t = half_transposed(b.pl[p], id0, id1);
    HalfBlock<1> const o = half_split<1>(t);
    r.pl[p] = o.pl[0];
  }
  return r;
}

}  // namespace dlmi
