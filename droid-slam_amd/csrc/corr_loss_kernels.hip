// Losses over the all-pairs correlation of feature maps, without the volume
// (the on-demand counterpart of CorrBlock, modules/corr.py:24-38,63-71, for
// training the features): for the edges e = (i, j) and the query pixels p of
// frame i
//   s_pq   = (scale / T) <f1[i][p], f2[j][q]>
//   loss_p = T^2 (sum_k pi_k log pi_k - sum_k pi_k s_p,idx(k) + log sum_q exp s_pq)
// with K sparse targets a row: one index, pi = 1, T = 1 (cross entropy), or a
// teacher's top logits, pi = softmax(t / T) (distillation).  With g = d/d loss:
//   ds_pq  = g_p T^2 (exp(s_pq - lse_p) - sum_{k: idx(k) = q} pi_k)
//   df1[i][p] += (scale / T) sum_q ds_pq f2[j][q]
//   df2[j][q] += (scale / T) sum_p ds_pq f1[i][p]
// summed over the edges a frame is in.
//
// The products run on MFMA 32x32x16 with the streamed frame as the A operand,
// so that a lane holds 16 streamed rows of ONE stationary row: the running
// maximum and sum of the softmax need no lane exchange until the very end, and
// the accumulator's layout is already the B operand's of the second product
// (its k slots (h, j) carry row 8 (j / 4) + 4 h + j % 4 of 16; the other
// operand comes by transposed LDS reads in the same order), so the weights ds
// never pass through LDS.
#include "lds_dma.hpp"

#include <algorithm>
#include <cmath>
#include <cstddef>

namespace droid {

namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));
typedef short short4_t __attribute__((vector_size(8)));

constexpr int kLT = 256;       // threads: 4 waves
constexpr int kRowsB = 128;    // stationary rows of a workgroup, 32 a wave
constexpr int kRowsY = 64;     // streamed rows a tile
constexpr int kMaxK = 64;      // sparse targets a row
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNegBig = -3.0e38f;   // running maximum before the first value (finite: no inf - inf)

template <typename T>
struct Op;
template <>
struct Op<_Float16> {
  typedef half8 vec8;
  static __device__ __forceinline__ floatx16 mfma(vec8 a, vec8 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Op<__bf16> {
  typedef bhalf8 vec8;
  static __device__ __forceinline__ floatx16 mfma(vec8 a, vec8 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

// A streamed tile in LDS: kRowsY rows of DP values, the 16-B slot s of row r
// stored at slot s ^ swz(r).  Rows of 256 B and more meet in the same banks, so
// r's low two bits move the slot by four and the next two by one: 16
// consecutive rows read at one slot (the first product) take 16 slots, and 4
// consecutive rows read at 4 slots (the transposed reads of the second) take
// 16 slots as well.  128-B rows: two share 256 B already.
template <int DP>
__device__ __forceinline__ int swz(int r) {
  if constexpr (DP == 64) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
  return ((r & 3) << 2) | ((r >> 2) & 3);
}

// LDS-DMA of rows y0 .. y0 + kRowsY - 1 of a frame (n rows of D values, descriptor
// rs over them); rows past n, slots past D and the rows that `skip` names land as zeros.
template <typename T, int DP, typename Skip>
__device__ __forceinline__ void stage_tile(rsrc_t rs, char* lds, int y0, int n, int D, int wave, int lane, Skip skip) {
  constexpr int RB = 2 * DP, NI = kRowsY * RB / 1024 / 4;
#pragma unroll
  for (int q = 0; q < NI; ++q) {
    const int o = (wave * NI + q) * 1024;
    const int row = (o + lane * 16) / RB, sl = (o + lane * 16) % RB / 16;
    const int s = sl ^ swz<DP>(row);
    const bool in = y0 + row < n && s * 8 < D && !skip(row);
    dma16(rs, lds_addr(lds) + o, in ? (unsigned)(((y0 + row) * D + s * 8) * 2) : kOob);
  }
}

// The stationary operand: lane (r = lane & 31, h = lane >> 5) holds values
// 16 k + 8 h .. + 7 of row x0 + r, zeros past the frame.
template <typename T, int DP>
__device__ __forceinline__ void load_rows(typename Op<T>::vec8 (&b)[DP / 16], const T* f, int x, int n, int D, int h) {
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) {
    const int d = 16 * k + 8 * h;
    if (x < n && d < D) b[k] = *reinterpret_cast<const typename Op<T>::vec8*>(f + (long)x * D + d);
    else b[k] = typename Op<T>::vec8{};
  }
}

// LDS byte address of lane (r = lane & 31, h)'s first 16 B of tile row r; its
// k-th pair of slots is at the address XOR (k << 5) (rows are aligned to their
// size), 32 rows further at + 32 rows.
template <int DP>
__device__ __forceinline__ unsigned row_addr(unsigned tile, int lane) {
  const int r = lane & 31, h = lane >> 5;
  return tile + r * 2 * DP + ((h ^ swz<DP>(r)) << 4);
}

// s[row of the tile's 32-row block][stationary row] = tile . stationary^T
template <typename T, int DP>
__device__ __forceinline__ floatx16 block_product(unsigned row0, int blk, const typename Op<T>::vec8 (&b)[DP / 16]) {
  typedef const __attribute__((address_space(3))) typename Op<T>::vec8* ptr;
  floatx16 acc;
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
#pragma unroll
  for (int k = 0; k < DP / 16; ++k)
    acc = Op<T>::mfma(*(ptr)(uintptr_t)((row0 ^ (k << 5)) + blk * 64 * DP), b[k], acc);
  return acc;
}

// v, as a value that the compiler knows nothing of: what is computed from it is
// computed here and not kept in registers over the loops around.
__device__ __forceinline__ int fresh(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// workgroup -> work item: the 8 XCDs each take a contiguous share, so the
// workgroups that stream the same frame share an L2.
__device__ __forceinline__ int xcd_item(int bid, int items) {
  const int per = (items + 7) / 8;
  return (bid & 7) * per + (bid >> 3);   // >= items: nothing to do
}

struct FwdArgs {
  const void *f1, *f2;
  const int *e1, *e2;          // (E) frame rows
  const int* idx;              // (E, P, K)
  float2* part;                // (E, P, S) running maximum (log2 units) and sum
  int E, N1, P, N2, Q, D, K, tiles, S, items;
  float c;                     // scale / T log2(e)
};

// Per query row the maximum and the sum of 2^(c s - max) over a share of the keys.
template <typename T, int DP>
__global__ void __launch_bounds__(kLT) corr_lse_kernel(FwdArgs a) {
  __shared__ __attribute__((aligned(1024))) char tile[2][kRowsY * 2 * DP];
  const int item = xcd_item(blockIdx.x, a.items);
  if (item >= a.items) return;
  const int s = item % a.S, pt = item / a.S % a.tiles, e = item / a.S / a.tiles;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = a.e1[e], j = a.e2[e];
  if (i < 0 || i >= a.N1 || j < 0 || j >= a.N2) return;   // the row kernel answers NaN
  const int p = pt * kRowsB + wave * 32 + (lane & 31);
  // rows without a target need no sum; a workgroup of them does nothing
  bool want = false;
  if (p < a.P)
    for (int k = 0; k < a.K; ++k) want |= a.idx[((long)e * a.P + p) * a.K + k] >= 0;
  if (!__syncthreads_or(want)) return;
  const T* f1 = static_cast<const T*>(a.f1) + (long)i * a.P * a.D;
  const T* f2 = static_cast<const T*>(a.f2) + (long)j * a.Q * a.D;
  const rsrc_t rs = make_rsrc(f2, (unsigned)a.Q * a.D * 2);
  const int nt = (a.Q + kRowsY - 1) / kRowsY;
  const int t0 = nt * s / a.S, t1 = nt * (s + 1) / a.S;
  typename Op<T>::vec8 b[DP / 16];
  load_rows<T, DP>(b, f1, p, a.P, a.D, lane >> 5);
  auto none = [](int) { return false; };
  stage_tile<T, DP>(rs, tile[0], t0 * kRowsY, a.Q, a.D, wave, lane, none);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  float m = kNegBig, l = 0.f;
  for (int t = t0; t < t1; ++t) {
    const unsigned row0 = row_addr<DP>(lds_addr(tile[(t - t0) & 1]), lane);
    if (t + 1 < t1) stage_tile<T, DP>(rs, tile[(t + 1 - t0) & 1], (t + 1) * kRowsY, a.Q, a.D, wave, lane, none);
    floatx16 sc[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) sc[k] = block_product<T, DP>(row0, k, b);
    if ((t + 1) * kRowsY > a.Q) {   // keys past the end
      const int y = t * kRowsY + 4 * (lane >> 5);
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int q = 0; q < 16; ++q)
          if (y + 32 * k + 8 * (q >> 2) + (q & 3) >= a.Q) sc[k][q] = -INFINITY;
    }
    float mx = sc[0][0];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int q = 0; q < 16; ++q) mx = fmaxf(mx, sc[k][q]);
    const float mn = fmaxf(m, mx * a.c);
    l *= __builtin_amdgcn_exp2f(m - mn);
    m = mn;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int q = 0; q < 16; ++q) l += __builtin_amdgcn_exp2f(fmaf(sc[k][q], a.c, -m));
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  }
  const float mo = __shfl_xor(m, 32, 64), lo = __shfl_xor(l, 32, 64);
  const float mm = fmaxf(m, mo);
  l = l * __builtin_amdgcn_exp2f(m - mm) + lo * __builtin_amdgcn_exp2f(mo - mm);
  if (lane < 32 && p < a.P) a.part[((long)e * a.P + p) * a.S + s] = make_float2(mm, l);
}

struct RowArgs {
  const void *f1, *f2;
  const int *e1, *e2, *idx;
  const float* logits;         // (E, P, K); null: cross entropy
  const float2* part;
  float *loss, *lse, *prob;    // (E, P), (E, P) log2 units, (E, P, K)
  int N1, P, N2, Q, D, K, S;
  long rows;
  float scale, invT, T2;
};

// One query row on 16 lanes: joins the shares of its sum, takes the K target
// logits as fp32 dot products (a row of D values is 16 lanes x 16 B) and forms
// the loss.  Rows without a target (all negative, or logits of -inf): loss 0 and lse = +inf, which
// makes every weight of the backward pass 0.  A target >= Q, an edge outside the
// frames: NaN.
template <typename T>
__global__ void __launch_bounds__(kLT) corr_loss_row_kernel(RowArgs a) {
  const long row = (long)blockIdx.x * (kLT / 16) + threadIdx.x / 16;
  const int l = threadIdx.x & 15;
  if (row >= a.rows) return;   // whole 16-lane groups
  const int e = (int)(row / a.P);
  const long p = row % a.P;
  const int i = a.e1[e], j = a.e2[e];
  const bool edge = i >= 0 && i < a.N1 && j >= 0 && j < a.N2;
  const int* idx = a.idx + row * a.K;
  auto sum16 = [](float v) {
#pragma unroll
    for (int o = 8; o; o >>= 1) v += __shfl_xor(v, o, 16);
    return v;
  };
  auto max16 = [](float v) {
#pragma unroll
    for (int o = 8; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 16));
    return v;
  };
  // the targets' weights: lane l has entries l, l + 16, ...
  float pi[kMaxK / 16];
  float top = -INFINITY;
  bool used = false, bad = !edge;
#pragma unroll
  for (int n = 0; n < kMaxK / 16; ++n) {
    pi[n] = -INFINITY;
    const int k = l + 16 * n;
    if (k < a.K) {
      const int t = idx[k];
      if (t >= 0) pi[n] = a.logits ? a.logits[row * a.K + k] * a.invT : 0.f;
      used |= pi[n] != -INFINITY;          // a logit of -inf: no target either
      bad |= t >= a.Q || pi[n] != pi[n];
      top = fmaxf(top, pi[n]);
    }
  }
  const float any = max16(used ? 1.f : 0.f), wrong = max16(bad ? 1.f : 0.f);
  if (any == 0.f || wrong != 0.f) {
    const bool ignored = any == 0.f;
    if (l == 0) {
      a.loss[row] = ignored ? 0.f : NAN;
      a.lse[row] = ignored ? INFINITY : NAN;
    }
    if (a.prob)
      for (int k = l; k < a.K; k += 16) a.prob[row * a.K + k] = 0.f;
    return;
  }
  top = max16(top);
  float tot = 0.f;
#pragma unroll
  for (int n = 0; n < kMaxK / 16; ++n) {
    pi[n] = __expf(pi[n] - top);
    if (l + 16 * n >= a.K) pi[n] = 0.f;
    tot += pi[n];
  }
  tot = sum16(tot);
  float ent = 0.f;
#pragma unroll
  for (int n = 0; n < kMaxK / 16; ++n) {
    pi[n] /= tot;
    if (pi[n] > 0.f) ent += pi[n] * logf(pi[n]);
    if (a.prob && l + 16 * n < a.K) a.prob[row * a.K + l + 16 * n] = pi[n];
  }
  // the row's sum over all keys
  float m = kNegBig;
  for (int s = l; s < a.S; s += 16) m = fmaxf(m, a.part[row * a.S + s].x);
  m = max16(m);
  float sum = 0.f;
  for (int s = l; s < a.S; s += 16) {
    const float2 v = a.part[row * a.S + s];
    sum += v.y * __builtin_amdgcn_exp2f(v.x - m);
  }
  sum = sum16(sum);
  const float lse2 = m + log2f(sum);
  // sum_k pi_k s_k, as one dot product with the pi-weighted sum of the target rows
  const T* f1 = static_cast<const T*>(a.f1) + ((long)i * a.P + p) * a.D;
  const T* f2 = static_cast<const T*>(a.f2) + (long)j * a.Q * a.D;
  float dot = 0.f;
  for (int k = 0; k < a.K; ++k) {
    const int t = idx[k];
    float w = 0.f;
#pragma unroll
    for (int n = 0; n < kMaxK / 16; ++n)
      if (k / 16 == n) w = __shfl(pi[n], k & 15, 16);
    if (t < 0 || w == 0.f) continue;
    float v = 0.f;
    for (int d = 8 * l; d < a.D; d += 128) {
      const auto x = *reinterpret_cast<const typename Op<T>::vec8*>(f1 + d);
      const auto y = *reinterpret_cast<const typename Op<T>::vec8*>(f2 + (long)t * a.D + d);
#pragma unroll
      for (int q = 0; q < 8; ++q) v = fmaf((float)x[q], (float)y[q], v);
    }
    dot = fmaf(w, v, dot);
  }
  dot = sum16(dot);
  ent = sum16(ent);
  if (l == 0) {
    a.loss[row] = a.T2 * (ent + fmaf(lse2, kLn2, -dot * (a.scale * a.invT)));
    a.lse[row] = lse2;
  }
}

// Largest |g| of an edge's rows (fp16: the weights are scaled by a power of two
// so that their largest is 2^13 .. 2^14 and the small ones stay normal numbers).
__global__ void __launch_bounds__(kLT) corr_gmax_kernel(const float* __restrict__ g, int P, float* __restrict__ out) {
  __shared__ float red[kLT / 64];
  float m = 0.f;
  for (int p = threadIdx.x; p < P; p += kLT) m = fmaxf(m, fabsf(g[(long)blockIdx.x * P + p]));
  for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) out[blockIdx.x] = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

struct BwdArgs {
  const void *f1, *f2;
  const int *e1, *e2, *idx;
  const float *prob, *lse, *g; // prob null: 1
  const float* gmax;           // (E), fp16 only
  void *d1, *d2;               // (N1, P, D), (N2, Q, D); shared: f1 and f2 are one tensor, d1 has both gradients
  float *part1, *part2;        // (S1, N1 P, D), (S2, N2 Q, D) where a gradient is made of several shares
  int E, N1, P, N2, Q, D, K, shared;
  int S1, S2, tiles1, tiles2;  // shares of the streamed rows; 128-row tiles a frame
  int items1, items;           // workgroups of d1 (0: not wanted), of d1 and d2
  float c, out_scale;          // scale / T log2(e); scale T
};

// Power of two that brings gmax to [2^13, 2^14)
__device__ __forceinline__ int g_exponent(float gmax) {
  if (!(gmax > 0.f) || gmax > 3.0e38f) return 0;
  int ex;
  frexpf(gmax, &ex);
  return max(-100, min(100, 14 - ex));
}

// What a workgroup of the gradient kernel keeps in LDS (dynamic: the sparse
// entries' part depends on K).
template <int DP>
struct BwdShared {
  char tile[2][kRowsY * 2 * DP];           // rows aligned to their size
  float delta[4][kRowsY][32];              // a wave's sparse terms of the current tile; zero between tiles
  float rowl[3][kRowsY], rowg[3][kRowsY];  // the streamed queries' lse and g, two tiles ahead
  int elist[kLT];
  int ecount[4];
  float redm[4];
  __attribute__((aligned(16))) int ent[1]; // 128 K sparse entries: a wave's rows each (SRC), two tiles (else)
};
template <int DP>
size_t bwd_lds(int K) {
  return offsetof(BwdShared<DP>, ent) + (size_t)kRowsB * K * sizeof(int);
}

// One edge e of the stationary frame: SRC: the rows x are its queries and the
// keys stream; otherwise x are its keys and the queries stream.  Tile by tile
// the logits are recomputed, turned into weights ds, and
// acc[d][x] += sum_y tile[y][d] ds[y][x].
//
// The sparse targets of a tile (pi at (y, x)) go through a dense, wave-private
// LDS image of the tile that is read only where one was put: the subtraction
// happens in fp32, before the rounding (p - pi of a well-trained row is a small
// difference).  To find them a wave compares its 32 rows' K entries (SRC, in LDS
// for the whole edge) or the tile's 64 K (staged with the tile) with the range
// it holds.
template <typename T, int DP, bool SRC>
__device__ __forceinline__ void bwd_edge(const BwdArgs& a, BwdShared<DP>& sh, int e, int split, int S, int R, int x0,
                                         float mul, const typename Op<T>::vec8 (&b)[DP / 16],
                                         floatx16 (&acc)[DP / 32]) {
  typedef typename Op<T>::vec8 vec8;
  typedef int int4_t __attribute__((ext_vector_type(4)));
  typedef int int4_u __attribute__((ext_vector_type(4), aligned(4)));
  constexpr int RB = 2 * DP, NI = kRowsY * RB / 1024 / 4;
  const int tid = fresh(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int xw = x0 + wave * 32, x = xw + (lane & 31);
  const int other = SRC ? a.e2[e] : a.e1[e];
  if (other < 0 || other >= (SRC ? a.N2 : a.N1)) return;
  const int n_y = SRC ? a.Q : a.P;
  const rsrc_t rs = make_rsrc(static_cast<const T*>(SRC ? a.f2 : a.f1) + (long)other * n_y * a.D,
                              (unsigned)n_y * a.D * 2);
  const int nt = (n_y + kRowsY - 1) / kRowsY;
  const int t0 = nt * split / S, t1 = nt * (split + 1) / S;
  if (t0 == t1) return;
  const float* lse = a.lse + (long)e * a.P;
  const float* g = a.g + (long)e * a.P;
  const int* idx = a.idx + (long)e * a.P * a.K;
  const float* prob = a.prob ? a.prob + (long)e * a.P * a.K : nullptr;
  const int K = a.K;
  float lx = INFINITY, gx = 0.f;
  if constexpr (SRC) {
    if (x < R) {
      lx = lse[x];
      gx = lx == INFINITY ? 0.f : lx == lx ? g[x] * mul : NAN;
    }
    if (!__syncthreads_or(lx != INFINITY)) return;   // every row left out: nothing here, whatever the keys hold
    for (int q = tid; q < kRowsB * K; q += kLT) sh.ent[q] = x0 + q / K < R ? idx[(long)x0 * K + q] : -1;
  }
  // Streamed queries: entries come one tile ahead, lse and g two: lse = +inf
  // marks a left-out row, whose features must not be read, before it is staged.
  float nl = 0.f, ng = 0.f;
  int4_t ne = {-1, -1, -1, -1};
  auto rows = [&](int t) {
    if (!SRC && tid < kRowsY) {
      const unsigned y = t * kRowsY + tid;
      nl = y < (unsigned)n_y ? lse[y] : INFINITY;
      ng = nl == INFINITY ? 0.f : nl == nl ? g[y] * mul : NAN;
    }
  };
  auto put_rows = [&](int slot) {
    if (!SRC && tid < kRowsY) {
      sh.rowl[slot][tid] = nl;
      sh.rowg[slot][tid] = ng;
    }
  };
  auto piece = [&](int t, int q) -> int4_t {   // entries 4 q .. + 3 of tile t
    const unsigned at = t * kRowsY * K + 4 * q;
    const int left = n_y * K - (int)at;
    int4_t v = {-1, -1, -1, -1};
    if (left >= 4) v = *reinterpret_cast<const int4_u*>(idx + at);
    else if (left > 0) {
      v.x = idx[at];
      if (left > 1) v.y = idx[at + 1];
      if (left > 2) v.z = idx[at + 2];
    }
    return v;
  };
  auto entries = [&](int t) {
    if (!SRC && tid < 16 * K) ne = piece(t, tid);   // K <= 16: all of them
  };
  auto put_entries = [&](int t, int buf) {
    if constexpr (!SRC) {
      int4_t* to = reinterpret_cast<int4_t*>(sh.ent + buf * kRowsY * K);
      if (tid < 16 * K) to[tid] = ne;
      for (int q = tid + kLT; q < 16 * K; q += kLT) to[q] = piece(t, q);
    }
  };
  int slot = 0;   // of tile t's row data
  auto stage = [&](int t, int buf, int sl) {
    stage_tile<T, DP>(rs, sh.tile[buf], t * kRowsY, n_y, a.D, wave, lane,
                      [&](int row) { return !SRC && sh.rowl[sl][row] == INFINITY; });
  };
  entries(t0);
  put_entries(t0, 0);
  rows(t0);
  put_rows(0);
  if (t0 + 1 < t1) rows(t0 + 1);
  put_rows(1);
  if constexpr (!SRC) __syncthreads();
  stage(t0, 0, 0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1, next = slot == 2 ? 0 : slot + 1, after = next == 2 ? 0 : next + 1;
    const unsigned cur = lds_addr(sh.tile[buf]), row0 = row_addr<DP>(cur, fresh(lane));
    if (t + 1 < t1) {
      stage(t + 1, buf ^ 1, next);
      entries(t + 1);
      if (t + 2 < t1) rows(t + 2);
    }
    // this tile's sparse terms
    const int base = SRC ? t * kRowsY : xw, n4 = SRC ? 8 * K : 16 * K;
    constexpr unsigned span = SRC ? kRowsY : 32;
    const int4_t* ent = reinterpret_cast<const int4_t*>(sh.ent + (SRC ? wave * 32 * K : buf * kRowsY * K));
    bool hit = false;
    for (int q = lane; q < n4; q += 64) {
      const int4_t v = ent[q] - base;
      hit |= (unsigned)v.x < span || (unsigned)v.y < span || (unsigned)v.z < span || (unsigned)v.w < span;
    }
    const bool any = __ballot(hit) != 0;
    float (&dl)[kRowsY][32] = sh.delta[wave];
    auto sparse = [&](bool put) {
      for (int q = lane; q < 4 * n4; q += 64) {
        const int v = reinterpret_cast<const int*>(ent)[q] - base;
        if ((unsigned)v < span) {
          const int row = q / K;
          float& c = SRC ? dl[v][row] : dl[row][v];
          if (put) atomicAdd(&c, prob ? prob[(long)(SRC ? xw : t * kRowsY) * K + q] : 1.f);
          else c = 0.f;
        }
      }
    };
    if (any) sparse(true);
    vec8 ds[4];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const floatx16 sc = block_product<T, DP>(row0, k, b);
      float pr[16], gr[16];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float4 l4, g4;
        if constexpr (!SRC) {
          l4 = *reinterpret_cast<const float4*>(&sh.rowl[slot][32 * k + 8 * q + 4 * h]);
          g4 = *reinterpret_cast<const float4*>(&sh.rowg[slot][32 * k + 8 * q + 4 * h]);
        } else {
          l4 = make_float4(lx, lx, lx, lx);
          g4 = make_float4(gx, gx, gx, gx);
        }
        const float lq[4] = {l4.x, l4.y, l4.z, l4.w}, gq[4] = {g4.x, g4.y, g4.z, g4.w};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          // clamped to [0, 1]: a NaN logit of a left-out row counts as 0
          pr[4 * q + u] =
              __builtin_amdgcn_fmed3f(__builtin_amdgcn_exp2f(fmaf(sc[4 * q + u], a.c, -lq[u])), 0.f, 1.f);
          gr[4 * q + u] = gq[u];
        }
      }
      if (any) {
        const int v = fresh(lane);
        const float* col = &dl[4 * (v >> 5)][v & 31];
#pragma unroll
        for (int q = 0; q < 16; ++q) pr[q] -= col[(32 * k + 8 * (q >> 2) + (q & 3)) * 32];
      }
#pragma unroll
      for (int q = 0; q < 16; ++q) ds[2 * k + (q >> 3)][q & 7] = (T)(gr[q] * pr[q]);
    }
    if (any) sparse(false);
    // second product: rows d of the transposed tile.  As the address lane 4 q + p
    // of its 16-lane group a lane points at row 16 k + 8 u + 4 h + q, values
    // 32 d + 16 ((lane >> 4) & 1) + 4 p .. + 3; d and u move the swizzled address by
    // an XOR, k and u by whole rows.
    {
      const int v = fresh(lane), q4 = ((v & 15) >> 2) + 4 * (v >> 5), s0 = 2 * ((v >> 4) & 1) + ((v >> 1) & 1);
      const unsigned tr0 = cur + q4 * RB + ((s0 ^ swz<DP>(q4)) << 4) + (v & 1) * 8;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          short4_t r4[2];
#pragma unroll
          for (int u = 0; u < 2; ++u)
            r4[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(uintptr_t)(
                (tr0 ^ (d << 6 | u << 5)) + (16 * k + 8 * u) * RB));
          struct { short4_t lo, hi; } both = {r4[0], r4[1]};
          acc[d] = Op<T>::mfma(__builtin_bit_cast(vec8, both), ds[k], acc[d]);
        }
      }
    }
    if (t + 1 < t1) put_entries(t + 1, buf ^ 1);
    if (t + 2 < t1) put_rows(after);
    slot = next;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  }
}

// The edges at frame n in one role, 256 at a time, in order.
template <typename T, int DP, bool SRC>
__device__ __forceinline__ void bwd_role(const BwdArgs& a, BwdShared<DP>& sh, int n, int split, int S, int R, int x0,
                                         float mul, const typename Op<T>::vec8 (&b)[DP / 16],
                                         floatx16 (&acc)[DP / 32]) {
  const int tid = fresh(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int* at_n = SRC ? a.e1 : a.e2;
  for (int e0 = 0; e0 < a.E; e0 += kLT) {
    const bool in = e0 + tid < a.E && at_n[e0 + tid] == n;
    const unsigned long long bal = __ballot(in);
    if (lane == 0) sh.ecount[wave] = __popcll(bal);
    __syncthreads();
    int at = __popcll(bal & ((1ull << lane) - 1));
    for (int q = 0; q < wave; ++q) at += sh.ecount[q];
    if (in) sh.elist[at] = e0 + tid;
    const int cnt = __builtin_amdgcn_readfirstlane(sh.ecount[0] + sh.ecount[1] + sh.ecount[2] + sh.ecount[3]);
    __syncthreads();
    for (int q = 0; q < cnt; ++q)
      bwd_edge<T, DP, SRC>(a, sh, __builtin_amdgcn_readfirstlane(sh.elist[q]), split, S, R, x0, mul, b, acc);
    __syncthreads();
  }
}

// The gradient of 128 rows x of one frame, over the edges in which the frame is
// the source (its rows are queries) and the target (its rows are keys), summed
// in registers and written once.
template <typename T, int DP>
__global__ void __launch_bounds__(kLT, DP <= 128 ? 2 : 1) corr_loss_bwd_kernel(BwdArgs a) {
  constexpr bool kScaled = !__is_same(T, __bf16);
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  BwdShared<DP>& sh = *reinterpret_cast<BwdShared<DP>*>(lds);
  const int item = xcd_item(blockIdx.x, a.items);
  if (item >= a.items) return;
  const bool second = item >= a.items1;              // rows of f2
  const int S = second ? a.S2 : a.S1, split = (second ? item - a.items1 : item) % S;
  const int w = (second ? item - a.items1 : item) / S, tiles = second ? a.tiles2 : a.tiles1;
  const int n = w / tiles, x0 = w % tiles * kRowsB;
  const int R = second ? a.Q : a.P;                  // rows of this frame
  const T* mine = static_cast<const T*>(second ? a.f2 : a.f1) + (long)n * R * a.D;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int x = x0 + wave * 32 + (lane & 31);
  typename Op<T>::vec8 b[DP / 16];
  load_rows<T, DP>(b, mine, x, R, a.D, h);
  floatx16 acc[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int q = 0; q < 16; ++q) acc[d][q] = 0.f;
  for (int q = lane; q < kRowsY * 32; q += 64) (&sh.delta[wave][0][0])[q] = 0.f;

  const bool is_src = !second, is_dst = second || a.shared;
  float mul = 1.f;
  int ex = 0;
  if constexpr (kScaled) {
    float gm = 0.f;
    for (int e = tid; e < a.E; e += kLT)
      if ((is_src && a.e1[e] == n) || (is_dst && a.e2[e] == n)) gm = fmaxf(gm, a.gmax[e]);
    for (int o = 32; o; o >>= 1) gm = fmaxf(gm, __shfl_xor(gm, o, 64));
    if (lane == 0) sh.redm[wave] = gm;
    __syncthreads();
    ex = g_exponent(fmaxf(fmaxf(sh.redm[0], sh.redm[1]), fmaxf(sh.redm[2], sh.redm[3])));
    mul = ldexpf(1.f, ex);
  }

  // the two roles one after the other: in one loop the compiler keeps both roles'
  // values in registers and spills
  if (is_src) bwd_role<T, DP, true>(a, sh, n, split, S, R, x0, mul, b, acc);
  if (is_dst) bwd_role<T, DP, false>(a, sh, n, split, S, R, x0, mul, b, acc);

  if (x >= R) return;
  const float out = a.out_scale * (kScaled ? ldexpf(1.f, -ex) : 1.f);
  const long row = (long)n * R + x;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int c = 32 * d + 8 * q + 4 * h;
      if (c >= a.D) continue;
      float v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = acc[d][4 * q + u] * out;
      if (S > 1) {
        float* part = (second ? a.part2 : a.part1) + (long)split * (second ? a.N2 : a.N1) * R * a.D;
        *reinterpret_cast<float4*>(part + row * a.D + c) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
        typedef T t4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<t4*>(static_cast<T*>(second ? a.d2 : a.d1) + row * a.D + c) =
            t4{(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
      }
    }
}

// dfmap = the sum of the S shares, in order
template <typename T>
__global__ void __launch_bounds__(kLT) corr_loss_join_kernel(const float* __restrict__ part, T* __restrict__ d,
                                                             long n, int S) {
  const long at = ((long)blockIdx.x * kLT + threadIdx.x) * 4;
  if (at >= n) return;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < S; ++s) {
    const float4 p = *reinterpret_cast<const float4*>(part + s * n + at);
    v.x += p.x;
    v.y += p.y;
    v.z += p.z;
    v.w += p.w;
  }
  typedef T t4 __attribute__((ext_vector_type(4)));
  *reinterpret_cast<t4*>(d + at) = t4{(T)v.x, (T)v.y, (T)v.z, (T)v.w};
}

// Shares of the streamed axis: enough workgroups for the 256 CUs, no more shares than tiles.
int fwd_split(int E, int P, int Q) {
  const long blocks = (long)E * ceil_div(P, kRowsB);
  return (int)std::max<long>(1, std::min<long>(ceil_div(Q, kRowsY), 1024 / std::max<long>(1, blocks)));
}

// The gradient's work split.  A workgroup's time is the tiles it streams (about
// E / N1 frames of Q / 64 tiles for a tile of f1's rows), and `slots` of them run
// at once; more shares even out the last round but write fp32 partial sums and
// read them back.  Takes the cheapest of the candidates in units of one tile's
// time (measured 2 us; 10 MB of partial sums at the copy rate).
struct BwdPlan {
  int tiles1, tiles2, S1, S2;
  long items1, items;
  size_t part1, part2;   // floats
};
BwdPlan bwd_plan(int E, int N1, int P, int N2, int Q, int D, bool shared) {
  BwdPlan b{};
  b.tiles1 = ceil_div(P, kRowsB), b.tiles2 = ceil_div(Q, kRowsB);
  const int yt1 = ceil_div(Q, kRowsY), yt2 = ceil_div(P, kRowsY);
  const double w1 = N1 ? (double)E / N1 * yt1 * (shared ? 2 : 1) : 0, w2 = N2 ? (double)E / N2 * yt2 : 0;
  const long n1 = (long)N1 * b.tiles1, n2 = (long)N2 * b.tiles2;
  const int slots = D <= 128 ? 512 : 256;
  const double per = (n1 * w1 + n2 * w2) / slots;   // tiles a slot
  double best = INFINITY;
  for (int r = 1; r <= 12; ++r) {
    const double grain = std::max(4.0, per / r);
    const int S1 = (int)std::min<double>(yt1, std::max(1.0, std::ceil(w1 / grain - 0.25)));
    const int S2 = (int)std::min<double>(yt2, std::max(1.0, std::ceil(w2 / grain - 0.25)));
    const long items = n1 * S1 + n2 * S2;
    const size_t p1 = S1 > 1 ? (size_t)S1 * N1 * P * D : 0, p2 = S2 > 1 ? (size_t)S2 * N2 * Q * D : 0;
    const double each = std::max(w1 / S1, w2 / S2) + 2.0;   // and two tiles' time to begin and end
    const double time = (items + slots - 1) / slots * each + (p1 + p2) * 8e-7;
    if (time < best) {
      best = time;
      b.S1 = S1, b.S2 = S2, b.part1 = p1, b.part2 = p2;
      b.items1 = n1 * S1, b.items = items;
    }
  }
  return b;
}

int corr_loss_check(const std::string& w, int dtype, int E, int N1, int P, int N2, int Q, int D, int K, float scale,
                    float T) {
  if (dtype != 0 && dtype != 3) return fail(kInvalidArgument, w + ": features must be float16 or bfloat16");
  if (E < 0 || N1 < 0 || N2 < 0 || P < 0 || Q <= 0 || D <= 0 || D % 8 || D > 256 || K < 1 || K > kMaxK)
    return fail(kInvalidArgument, w + ": bad arguments (Q > 0, 0 < D <= 256, D % 8 == 0, 1 <= K <= 64)");
  if (!(scale > 0.f) || !std::isfinite(scale) || !(T > 0.f) || !std::isfinite(T))
    return fail(kInvalidArgument, w + ": scale and temperature must be positive and finite");
  if ((long)std::max(P, Q) * D * 2 > 0x7fffffffL || (long)P * K > 0x1fffffffL || (long)E * std::max(1, ceil_div(P, kRowsB)) > 0x3fffffL ||
      (long)(N1 + (long)N2) * ceil_div(std::max(P, Q), kRowsB) > 0x3fffffL)
    return fail(kUnsupported, w + ": maps too large");
  return kOk;
}

size_t gmax_bytes(int E) { return ((size_t)E * sizeof(float) + 15) / 16 * 16; }

bool unaligned(const void* p) { return reinterpret_cast<uintptr_t>(p) & 15; }

}  // namespace

}  // namespace droid

using namespace droid;

#define CORR_DIMS(T, LAUNCH) \
  if (D <= 64) { LAUNCH(T, 64); } else if (D <= 128) { LAUNCH(T, 128); } else { LAUNCH(T, 256); }
#define CORR_TYPES(LAUNCH) \
  if (dtype == 0) { CORR_DIMS(_Float16, LAUNCH) } else { CORR_DIMS(__bf16, LAUNCH) }

extern "C" {

size_t droid_corr_loss_workspace(int E, int N1, int P, int N2, int Q, int D, int shared, int backward) {
  if (E <= 0 || N1 < 0 || P <= 0 || N2 < 0 || Q <= 0 || D <= 0) return 0;
  if (!backward) return (size_t)E * P * fwd_split(E, P, Q) * sizeof(float2);
  const BwdPlan b = bwd_plan(E, N1, P, N2, Q, D, shared);
  return gmax_bytes(E) + (b.part1 + b.part2) * sizeof(float);
}

int droid_corr_loss_forward(int dtype, const void* fmap1, const void* fmap2, const int* f1, const int* f2,
                            const int* idx, const float* logits, float* loss, float* lse, float* prob, int E, int N1,
                            int P, int N2, int Q, int D, int K, float scale, float temperature, void* ws,
                            size_t ws_bytes, hipStream_t stream) {
  const std::string what = "corr_loss_forward";
  if (const int st = corr_loss_check(what, dtype, E, N1, P, N2, Q, D, K, scale, temperature)) return st;
  if (E == 0 || P == 0) return kOk;
  if (!fmap1 || !fmap2 || !f1 || !f2 || !idx || !loss || !lse || (logits && !prob))
    return fail(kInvalidArgument, what + ": null tensor");
  if (!logits && K != 1) return fail(kInvalidArgument, what + ": one target a row without logits");
  if (unaligned(fmap1) || unaligned(fmap2)) return fail(kInvalidArgument, what + ": features must be 16-B aligned");
  if (!ws || ws_bytes < droid_corr_loss_workspace(E, N1, P, N2, Q, D, 0, 0))
    return fail(kInvalidArgument, what + ": workspace too small");
  FwdArgs a{fmap1, fmap2, f1, f2, idx, static_cast<float2*>(ws), E, N1, P, N2, Q, D, K, ceil_div(P, kRowsB),
            fwd_split(E, P, Q), 0, scale / temperature * kLog2e};
  a.items = E * a.tiles * a.S;
#define LSE(T, DP) corr_lse_kernel<T, DP><<<(a.items + 7) / 8 * 8, kLT, 0, stream>>>(a)
  CORR_TYPES(LSE)
#undef LSE
  DROID_LAUNCH_CHECK();
  RowArgs r{fmap1, fmap2, f1, f2, idx, logits, a.part, loss, lse, logits ? prob : nullptr, N1, P, N2, Q, D, K, a.S,
            (long)E * P, scale, 1.f / temperature, temperature * temperature};
  const int grid = (int)((r.rows + kLT / 16 - 1) / (kLT / 16));
  if (dtype == 0) corr_loss_row_kernel<_Float16><<<grid, kLT, 0, stream>>>(r);
  else corr_loss_row_kernel<__bf16><<<grid, kLT, 0, stream>>>(r);
  DROID_LAUNCH_CHECK();
  return kOk;
}

int droid_corr_loss_backward(int dtype, const void* fmap1, const void* fmap2, const int* f1, const int* f2,
                             const int* idx, const float* prob, const float* lse, const float* gloss, void* dfmap1,
                             void* dfmap2, int shared, int E, int N1, int P, int N2, int Q, int D, int K, float scale,
                             float temperature, void* ws, size_t ws_bytes, hipStream_t stream) {
  const std::string what = "corr_loss_backward";
  if (const int st = corr_loss_check(what, dtype, E, N1, P, N2, Q, D, K, scale, temperature)) return st;
  if (E == 0 || P == 0) return fail(kInvalidArgument, what + ": no edges or no queries");
  if (!fmap1 || !fmap2 || !f1 || !f2 || !idx || !lse || !gloss || (!dfmap1 && !dfmap2))
    return fail(kInvalidArgument, what + ": null tensor");
  if (!prob && K != 1) return fail(kInvalidArgument, what + ": one target a row without weights");
  if (shared && (fmap1 != fmap2 || N1 != N2 || P != Q || dfmap2))
    return fail(kInvalidArgument, what + ": one shared feature tensor has one gradient");
  if (unaligned(fmap1) || unaligned(fmap2)) return fail(kInvalidArgument, what + ": features must be 16-B aligned");
  // the gradients that are wanted; a shared tensor's rows are counted once
  const int n1 = dfmap1 ? N1 : 0, n2 = dfmap2 ? N2 : 0;
  if (!ws || ws_bytes < droid_corr_loss_workspace(E, n1, P, n2, Q, D, shared, 1))
    return fail(kInvalidArgument, what + ": workspace too small");
  const BwdPlan b = bwd_plan(E, n1, P, n2, Q, D, shared != 0);
  if (b.items == 0) return kOk;
  if (b.items > 0x3fffffffL) return fail(kUnsupported, what + ": maps too large");
  float* gmax = static_cast<float*>(ws);
  BwdArgs a{};
  a.f1 = fmap1, a.f2 = fmap2, a.e1 = f1, a.e2 = f2, a.idx = idx, a.prob = prob, a.lse = lse, a.g = gloss;
  a.gmax = gmax, a.d1 = dfmap1, a.d2 = dfmap2;
  a.part1 = reinterpret_cast<float*>(static_cast<char*>(ws) + gmax_bytes(E)), a.part2 = a.part1 + b.part1;
  a.E = E, a.N1 = N1, a.P = P, a.N2 = N2, a.Q = Q, a.D = D, a.K = K, a.shared = shared != 0;
  a.S1 = b.S1, a.S2 = b.S2, a.tiles1 = b.tiles1, a.tiles2 = b.tiles2;
  a.items1 = (int)b.items1, a.items = (int)b.items;
  a.c = scale / temperature * kLog2e, a.out_scale = scale * temperature;
  if (dtype == 0) {
    corr_gmax_kernel<<<E, kLT, 0, stream>>>(gloss, P, gmax);
    DROID_LAUNCH_CHECK();
  }
  const int grid = (a.items + 7) / 8 * 8;
#define BWD(T, DP) corr_loss_bwd_kernel<T, DP><<<grid, kLT, bwd_lds<DP>(K), stream>>>(a)
  CORR_TYPES(BWD)
#undef BWD
  DROID_LAUNCH_CHECK();
  for (int q = 0; q < 2; ++q) {
    if (!(q ? b.part2 : b.part1)) continue;
    const long n = q ? (long)N2 * Q * D : (long)N1 * P * D;
    const float* part = q ? a.part2 : a.part1;
    const int jg = (int)((n / 4 + kLT - 1) / kLT), S = q ? a.S2 : a.S1;
    if (dtype == 0) corr_loss_join_kernel<_Float16><<<jg, kLT, 0, stream>>>(part, (_Float16*)(q ? dfmap2 : dfmap1), n, S);
    else corr_loss_join_kernel<__bf16><<<jg, kLT, 0, stream>>>(part, (__bf16*)(q ? dfmap2 : dfmap1), n, S);
    DROID_LAUNCH_CHECK();
  }
  return kOk;
}

}  // extern "C"
