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
// never pass through LDS.  The weights are rounded to the features' type for that
// product, after the sparse terms are subtracted in fp32, and fp16 ones are scaled
// by a power of two per frame.  Half tiles with a target take what the rounding left
// in a second product: a target's weight is most of its row's, and its half a step
// alone made the gradient's error 1.2 to 1.45 times that of rounding the result
// (it costs four clips 603 -> 613 us, 501 points 273 -> 300); elsewhere the weights are
// probabilities, and half a step of them is nothing beside that.
//
// What bounds it: the matrix instructions, at the 1.11 (fp16) to 1.16 (bf16) PFLOP/s
// that a large library product reaches on this card, with the exponentials' vector
// work beside them.  Four clips (96 edges of 2560 x 2560 rows, D = 128, bf16): row
// sums 162 us (161 GFLOP, 0.99 PFLOP/s), losses 33 us, gradient 385 us (349 GFLOP,
// 0.91 PFLOP/s) and 34 us beside it, 614 in all; one clip in fp16 50 + 11 + 134 + 28.
// (100 calls after another.  The comparisons in the comments below are of 15 calls,
// whose clock is lower: the gradient of 383 us before the second product of the
// remainder took 438 there.)
#include "lds_dma.hpp"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

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

// lds_dma.hpp's dma16_late with 4 B a lane.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma4(rsrc_t rs, unsigned lds, unsigned voff) {
  const rsrc_t r = {__builtin_amdgcn_readfirstlane(rs.x), __builtin_amdgcn_readfirstlane(rs.y),
                    __builtin_amdgcn_readfirstlane(rs.z), __builtin_amdgcn_readfirstlane(rs.w)};
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(r)
               : "memory", "m0");
}
#pragma clang diagnostic pop

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

// LDS-DMA of rows y0 .. y0 + kRowsY - 1 of a frame (n rows of D values): a lane's
// source within the tile does not depend on the tile (`off`: kOob past D), the
// descriptor starts at the tile's first row and ends with the frame, so that rows
// past it land as zeros; no vector instruction a load.
template <int DP>
constexpr int kDmas = kRowsY * 2 * DP / 4096;   // a wave
template <int DP>
__device__ __forceinline__ void lane_offsets(unsigned (&off)[kDmas<DP>], int D, int wave, int lane) {
  constexpr int RB = 2 * DP;
#pragma unroll
  for (int q = 0; q < kDmas<DP>; ++q) {
    const int o = (wave * kDmas<DP> + q) * 1024 + lane * 16, row = o / RB, s = (o % RB / 16) ^ swz<DP>(row);
    off[q] = s * 8 < D ? (unsigned)(row * D + s * 8) * 2 : kOob;
  }
}
template <typename T, int DP, typename Skip>
__device__ __forceinline__ void stage_tile(const T* frame, char* lds, int y0, int n, int D,
                                           const unsigned (&off)[kDmas<DP>], int wave, int lane, Skip skip) {
  const rsrc_t rs = make_rsrc(frame + (long)y0 * D, (unsigned)(n - y0) * D * 2);
#pragma unroll
  for (int q = 0; q < kDmas<DP>; ++q) {
    const int o = (wave * kDmas<DP> + q) * 1024;
    dma16_late(rs, lds_addr(lds) + o, skip((o + lane * 16) / (2 * DP)) ? kOob : off[q]);
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

// All of the wave's loads have landed, LDS-DMA included.  The builtin, not inline
// asm: the compiler does not count the DMAs, and where it cannot see that its own
// loads have landed it waits for "them" - in fact the DMAs in flight - again in
// every turn of the loop that follows.
__device__ __forceinline__ void loads_done() {
  __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
  asm volatile("" ::: "memory");
}

// The same, but for the wave's last N LDS-DMAs.
template <int N>
__device__ __forceinline__ void loads_left() {
  __builtin_amdgcn_s_waitcnt(0x0f70 | N);
  asm volatile("" ::: "memory");
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

// 32-row blocks of queries a wave: two where the registers allow three such
// workgroups a CU, since every operand read from shared memory then feeds two matrix
// instructions (with one, 128 B a clock of shared memory are as busy as they: four
// clips 178 us, with two 171; accumulators in AGPRs, copied out, 183).
template <int DP>
constexpr int kXF = DP <= 128 ? 2 : 1;
inline int fwd_rows(int D) { return D <= 128 ? 2 * kRowsB : kRowsB; }
inline int fwd_groups(int D) { return D <= 128 ? 3 : 2; }   // workgroups a CU

// Per query row the maximum and the sum of 2^(c s - max) over a share of the keys.
template <typename T, int DP>
__global__ void __launch_bounds__(kLT, DP <= 128 ? 3 : 2) corr_lse_kernel(FwdArgs a) {
  typedef const __attribute__((address_space(3))) typename Op<T>::vec8* ptr;
  constexpr int XF = kXF<DP>;
  __shared__ __attribute__((aligned(1024))) char tile[2][kRowsY * 2 * DP];
  const int item = xcd_item(blockIdx.x, a.items);
  if (item >= a.items) return;
  const int s = item % a.S, pt = item / a.S % a.tiles, e = item / a.S / a.tiles;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = a.e1[e], j = a.e2[e];
  if (i < 0 || i >= a.N1 || j < 0 || j >= a.N2) return;   // the row kernel answers NaN
  const int p0 = (pt * 4 + wave) * 32 * XF;
  // rows without a target need no sum; a workgroup of them does nothing
  bool want = false;
  if (p0 + lane < a.P && lane < 32 * XF)
    for (int k = 0; k < a.K; ++k) want |= a.idx[((long)e * a.P + p0 + lane) * a.K + k] >= 0;
  if (!__syncthreads_or(want)) return;
  const T* f1 = static_cast<const T*>(a.f1) + (long)i * a.P * a.D;
  const T* f2 = static_cast<const T*>(a.f2) + (long)j * a.Q * a.D;
  unsigned off[kDmas<DP>];
  lane_offsets<DP>(off, a.D, wave, lane);
  const int nt = (a.Q + kRowsY - 1) / kRowsY;
  const int t0 = nt * s / a.S, t1 = nt * (s + 1) / a.S;
  auto none = [](int) { return false; };
  stage_tile<T, DP>(f2, tile[0], t0 * kRowsY, a.Q, a.D, off, wave, lane, none);
  typename Op<T>::vec8 b[XF][DP / 16];
#pragma unroll
  for (int x = 0; x < XF; ++x) load_rows<T, DP>(b[x], f1, p0 + 32 * x + (lane & 31), a.P, a.D, lane >> 5);
  loads_done();
  __syncthreads();
  float m[XF], l[XF];
#pragma unroll
  for (int x = 0; x < XF; ++x) m[x] = kNegBig, l[x] = 0.f;
  for (int t = t0; t < t1; ++t) {
    const unsigned row0 = row_addr<DP>(lds_addr(tile[(t - t0) & 1]), lane);
    if (t + 1 < t1) stage_tile<T, DP>(f2, tile[(t + 1 - t0) & 1], (t + 1) * kRowsY, a.Q, a.D, off, wave, lane, none);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      floatx16 sc[XF];
#pragma unroll
      for (int x = 0; x < XF; ++x)
#pragma unroll
        for (int q = 0; q < 16; ++q) sc[x][q] = 0.f;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) {
        const typename Op<T>::vec8 f = *(ptr)(uintptr_t)((row0 ^ (d << 5)) + k * 64 * DP);
#pragma unroll
        for (int x = 0; x < XF; ++x) sc[x] = Op<T>::mfma(f, b[x][d], sc[x]);
      }
      if (t * kRowsY + 32 * k + 32 > a.Q) {   // keys past the end
        const int y = t * kRowsY + 32 * k + 4 * (lane >> 5);
#pragma unroll
        for (int x = 0; x < XF; ++x)
#pragma unroll
          for (int q = 0; q < 16; ++q)
            if (y + 8 * (q >> 2) + (q & 3) >= a.Q) sc[x][q] = -INFINITY;
      }
#pragma unroll
      for (int x = 0; x < XF; ++x) {
        float mx = sc[x][0];
#pragma unroll
        for (int q = 1; q < 16; ++q) mx = fmaxf(mx, sc[x][q]);
        const float mn = fmaxf(m[x], mx * a.c);
        l[x] *= __builtin_amdgcn_exp2f(m[x] - mn);
        m[x] = mn;
#pragma unroll
        for (int q = 0; q < 16; ++q) l[x] += __builtin_amdgcn_exp2f(fmaf(sc[x][q], a.c, -mn));
      }
    }
    loads_done();
    __syncthreads();
  }
#pragma unroll
  for (int x = 0; x < XF; ++x) {
    const float mo = __shfl_xor(m[x], 32, 64), lo = __shfl_xor(l[x], 32, 64);
    const float mm = fmaxf(m[x], mo);
    const float sum = l[x] * __builtin_amdgcn_exp2f(m[x] - mm) + lo * __builtin_amdgcn_exp2f(mo - mm);
    const int p = p0 + 32 * x + (lane & 31);
    if (lane < 32 && p < a.P) a.part[((long)e * a.P + p) * a.S + s] = make_float2(mm, sum);
  }
}

struct RowArgs {
  const void *f1, *f2;
  const int *e1, *e2, *idx;
  const float* logits;         // (E, P, K); null: cross entropy
  const float2* part;
  float *loss, *lse, *prob;    // (E, P), (E, P) log2 units, (E, P, K)
  int N1, P, N2, Q, D, K, S;
  long rows;
  float invT, T2, c;           // c: scale / T log2(e)
};

// One query row on 16 lanes: joins the shares of its sum, takes the K target
// logits as fp32 dot products (a row of D values is 16 lanes x 16 B) and forms
// the loss.  Rows without a target (all negative, or logits of -inf): loss 0 and
// lse = +inf, or -inf where the row's features are not all finite (the backward
// pass must not touch those).  A target >= Q, an edge outside the frames: NaN.
// SLOTS: targets a lane holds (K <= 16 SLOTS); kBatch: target rows read at once.
// Bound by the rows it gathers, 256 B each, mostly from L2: 246 thousand queries
// with one target 36 us (as <4, 4>: 57), with 16 100 us (10 TB/s; as <4, 4> 131,
// one row at a time 155); 33 and 92 in a long run.
template <typename T, int SLOTS, int kBatch>
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
  float pi[SLOTS];
  int own[SLOTS];
  float top = -INFINITY;
  bool used = false, bad = !edge;
#pragma unroll
  for (int n = 0; n < SLOTS; ++n) {
    pi[n] = -INFINITY;
    own[n] = -1;
    const int k = l + 16 * n;
    if (k < a.K) {
      const int t = own[n] = idx[k];
      if (t >= 0) pi[n] = a.logits ? a.logits[row * a.K + k] : 0.f;
      used |= pi[n] != -INFINITY;          // a logit of -inf: no target either
      bad |= t >= a.Q || pi[n] != pi[n];
      top = fmaxf(top, pi[n]);
    }
  }
  const float any = max16(used ? 1.f : 0.f), wrong = max16(bad ? 1.f : 0.f);
  const T* f1 = static_cast<const T*>(a.f1) + ((long)i * a.P + p) * a.D;
  if (any == 0.f || wrong != 0.f) {
    const bool ignored = any == 0.f;
    float finite = 0.f;   // 0 while every feature is
    if (ignored && edge)
      for (int d = 8 * l; d < a.D; d += 128) {
        const auto x = *reinterpret_cast<const typename Op<T>::vec8*>(f1 + d);
#pragma unroll
        for (int q = 0; q < 8; ++q) finite = fmaf((float)x[q], 0.f, finite);
      }
    finite = sum16(finite);
    if (l == 0) {
      a.loss[row] = ignored ? 0.f : NAN;
      a.lse[row] = !ignored ? NAN : finite == 0.f ? INFINITY : -INFINITY;
    }
    if (a.prob)
      for (int k = l; k < a.K; k += 16) a.prob[row * a.K + k] = 0.f;
    return;
  }
  top = max16(top);
  float tot = 0.f;
#pragma unroll
  for (int n = 0; n < SLOTS; ++n) {
    // over T last: a lowest value over T < 1 is -inf.  The hardware's exponential: off by
    // t 2^-24 and two units of fp32 for an exponent -t, whose weight is e^-t of the largest
    pi[n] = __expf((pi[n] - top) * a.invT);
    if (l + 16 * n >= a.K) pi[n] = 0.f;
    tot += pi[n];
  }
  tot = sum16(tot);
  float ent = 0.f;
#pragma unroll
  for (int n = 0; n < SLOTS; ++n) {
    pi[n] /= tot;
    if (pi[n] > 0.f) ent += pi[n] * logf(pi[n]);
    if (pi[n] == 0.f) own[n] = -1;   // no target: a later place of its key may have weight
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
  const float over = sum > 0.f ? log2f(sum) : NAN, lse2 = m + over;
  // sum_k pi_k s_k, as one dot product with the pi-weighted sum of the target rows
  const T* f2 = static_cast<const T*>(a.f2) + (long)j * a.Q * a.D;
  // The weights kept for the gradient: a key that a row names more than once has all
  // of its weight at the first place that has any, so that no place of ds has more than
  // one term of an edge (and their sum no order).
  double dot = 0.0;
  float kept[SLOTS] = {};
  bool again[SLOTS] = {};
  typedef typename Op<T>::vec8 vec8;
  vec8 x[2] = {};             // the row's values 8 l .. + 7, and 128 further
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (8 * l + 128 * h < a.D) x[h] = *reinterpret_cast<const vec8*>(f1 + 8 * l + 128 * h);
  for (int k0 = 0; k0 < a.K; k0 += kBatch) {
    int t[kBatch];
    float w[kBatch];
    vec8 y[kBatch][2];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      t[u] = -1, w[u] = 0.f;
#pragma unroll
      for (int n = 0; n < SLOTS; ++n)   // (a lane past K holds -1 and 0)
        if (k0 / 16 == n) t[u] = __shfl(own[n], (k0 + u) & 15, 16), w[u] = __shfl(pi[n], (k0 + u) & 15, 16);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (t[u] >= 0 && 8 * l + 128 * h < a.D)
          y[u][h] = *reinterpret_cast<const vec8*>(f2 + (long)t[u] * a.D + 8 * l + 128 * h);
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (t[u] < 0) continue;
      if (a.prob) {
#pragma unroll
        for (int n = 0; n < SLOTS; ++n)
          if (16 * n < a.K) {
            again[n] |= own[n] == t[u] && k0 + u < l + 16 * n;
            kept[n] += own[n] == t[u] ? w[u] : 0.f;
          }
      }
      // (products of two features are exact in fp32; added as a tree: fewer roundings)
      float v = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (8 * l + 128 * h < a.D) {
          float p[4];
#pragma unroll
          for (int q = 0; q < 4; ++q)
            p[q] = fmaf((float)x[h][q], (float)y[u][h][q], (float)x[h][q + 4] * (float)y[u][h][q + 4]);
          v += (p[0] + p[2]) + (p[1] + p[3]);
        }
      dot = fma((double)w[u], (double)v, dot);
    }
  }
  if (a.prob) {
#pragma unroll
    for (int n = 0; n < SLOTS; ++n)
      if (l + 16 * n < a.K) a.prob[row * a.K + l + 16 * n] = again[n] ? 0.f : kept[n];
  }
#pragma unroll
  for (int o = 8; o; o >>= 1) dot += __shfl_xor(dot, o, 16);
  ent = sum16(ent);
  if (l == 0) {
    // lse - sum_k pi_k s_k relative to the largest logit m: where a target is near it
    // the loss is a small difference, whose rounding would be m's
    a.loss[row] = a.T2 * fmaf(over + (float)((double)m - dot * (double)a.c), kLn2, ent);
    a.lse[row] = lse2;
  }
}

// ---- the gradient -----------------------------------------------------------
//
// A work item is 256 rows x of one frame (128 where D > 128), held in registers; its steps are the
// 64-row tiles y of the frames that share an edge with it, streamed through LDS:
// the logits s[y][x] are recomputed, turned into weights
//   ds = g1[x] (p1 - pi1) + g2[y] (p2 - pi2)
// (1: an edge in which x are the queries and y keys, 2: one in which y are the
// queries), and acc[d][x] += sum_y tile[y][d] ds[y][x].  An edge (i, j) of one
// feature tensor is done together with its reverse (j, i), where the graph has
// it: both need the same logits and the same second product.
//
// The steps of all items, end to end, are cut into equal shares, one for each
// workgroup that the chip holds at once; an item that a cut goes through is
// summed from fp32 parts, in order, by the join kernel.  (Items of their own
// workgroup each left half the chip idle in the last round: 560 items on 512
// places took 1137 us, shares of the streamed axis by a cost model 867 us, with
// uneven graphs up to twice their even share.)
//
// One workgroup a CU, one wave a SIMD with all 512 registers, so the order of a
// step's instructions is written out: matrix instructions between the exponentials,
// shared memory read between matrix instructions, the last second product of a tile
// in the next step.  A step of a pair takes 5200 clocks for 2048 of matrix
// instructions (512 more in a half tile with targets); the rest is the exponentials (32 a lane and half, 8 clocks each),
// the conversion to 16 bits, accumulators copied out of AGPRs, two waits at the barrier
// (480) and the tile's loads.  On the way, four clips: 32 rows a wave 531 us, 64
// rows 522, the sparse terms sorted beforehand 479, one exponential for both
// directions and this order 455, the streamed factor made once a workgroup 438.

constexpr int kUnitBoth = 5, kUnitSrc = 4, kUnitDst = 4;   // relative cost of a step (measured 5670 : 4460 : 4380 clk)
// Rows x of a wave, in 32s.  Two where their accumulators fit the registers of one
// wave a SIMD: a tile read from LDS then serves twice the products.  With one (two
// waves a SIMD) the LDS pipe bound the kernel: four clips 508 us, the same without
// exponentials 511 us, without the second product 347 us.
template <int DP>
constexpr int kXH = DP <= 128 ? 2 : 1;
constexpr int bwd_rows(int D) { return 128 * (D <= 128 ? 2 : 1); }
constexpr int kJoin = 8;                     // workgroups that join one item
constexpr int kET = 1024;                    // threads of the edge kernel
constexpr float kRange = 40.f;                // see edge_paired
constexpr int kMaxGroups = 8192;             // of 64 keys: frames of up to 524288 rows
constexpr int kMaxEdges = 65536;             // between as many frames of one row 93 ms, growing with the square
constexpr int kMinUnits = 32;                // smallest share worth a workgroup

struct BwdArgs {
  const void *f1, *f2;
  const int *e1, *e2, *idx;
  const float *prob, *lse, *g; // prob null: 1
  void *d1, *d2;               // (N1, P, D), (N2, Q, D)
  float* gmax;                 // (E) largest |g|; -1: no row has a target
  int* flags;                  // (E) 1: a left-out row is not finite, 2: a g is negative
  float2* range;               // (E) smallest and largest lse of the rows with a target
  int* first_rec;              // (E, groups + 1) the records of each 64 keys
  uint2* rec;                  // (E, P K) query row << 6 | key & 63, and g pi
  float* expn;                 // (E, tiles of P, 64) the queries' exponents: log2 |g| - lse, -inf: no gradient
  int* partner;                // (E) the reverse edge that is done together with this one, -1: none
  long long* first;            // (V + 1) units before frame slot v; the slots: f1's frames (d1 wanted), then f2's
  int* expo;                   // (V) fp16: exponent that scales the slot's weights
  float* part;                 // (G, 2, 128, D)
  int E, N1, P, N2, Q, D, K, shared;
  int tiles1, tiles2;          // items of a frame (bwd_rows rows each)
  int n1, V, G;                // slots of f1, all slots, workgroups
  int groups;                  // of 64 keys a frame
  float c, out_scale;          // scale / T log2(e); scale T
};

__host__ __device__ __forceinline__ int y_tiles(int rows) { return (rows + kRowsY - 1) / kRowsY; }

// Power of two that brings gmax to [2^13, 2^14): an fp16 weight's largest value
// stays far from 65504 and the small ones stay normal numbers.
__device__ __forceinline__ int g_exponent(float gmax) {
  if (!(gmax > 0.f) || gmax > 3.0e38f) return 0;
  int ex;
  frexpf(gmax, &ex);
  return max(-100, min(100, 14 - ex));
}

// (96 edges of 2560 rows: 13 us with one target a row, 35 with 16 - one term read at
// a time 59 -, sorted anew by every workgroup of the gradient kernel 500 in all.)
// One workgroup an edge: what the gradient kernel wants of its rows, its sparse
// terms by 64 keys (a counting sort), and the reverse edge it may be paired with
// (the k-th copy of (i, j) with the k-th of (j, i)).
__global__ void __launch_bounds__(kET) corr_edge_kernel(BwdArgs a) {
  constexpr int kLT = kET;
  __shared__ float red[kLT / 64];
  __shared__ int cnt[kLT / 64], fl[kLT / 64];
  __shared__ float2 lr[kLT / 64];
  __shared__ int bucket[kMaxGroups];
  const int e = blockIdx.x, tid = threadIdx.x, wave = tid >> 6;
  const int padded = y_tiles(a.P) * kRowsY;
  float m = -1.f, lmin = INFINITY, lmax = -INFINITY;
  int f = 0;
  for (int p = tid; p < padded; p += kLT) {
    const float l = p < a.P ? a.lse[(long)e * a.P + p] : INFINITY;
    float v = -INFINITY;
    if (fabsf(l) != INFINITY) {
      const float g = a.g[(long)e * a.P + p];
      m = fmaxf(fmaxf(m, 0.f), fabsf(g));
      v = log2f(fabsf(g)) - l;
      lmin = fminf(lmin, l), lmax = fmaxf(lmax, l);
      if (g < 0.f) f |= 2;
    } else if (l < 0.f) {
      f |= 1;
    }
    a.expn[(long)e * padded + p] = v;
  }
  for (int o = 32; o; o >>= 1) {
    m = fmaxf(m, __shfl_xor(m, o, 64));
    f |= __shfl_xor(f, o, 64);
    lmin = fminf(lmin, __shfl_xor(lmin, o, 64));
    lmax = fmaxf(lmax, __shfl_xor(lmax, o, 64));
  }
  if ((tid & 63) == 0) red[wave] = m, fl[wave] = f, lr[wave] = make_float2(lmin, lmax);
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kLT / 64; ++w) {   // (this thread holds the first wave's)
      m = fmaxf(m, red[w]), f |= fl[w];
      lmin = fminf(lmin, lr[w].x), lmax = fmaxf(lmax, lr[w].y);
    }
    a.gmax[e] = m;
    a.flags[e] = f;
    a.range[e] = make_float2(lmin, lmax);
    a.partner[e] = -1;
  }
  // The records.  Their order within a bucket is that of the atomics: a place (y, x)
  // has at most one of an edge (corr_loss_row_kernel), one more of its reverse, and
  // their sum has no order.  More keys than buckets: a
  // bucket holds several groups, told apart by the reader (rec holds the key's low
  // bits only), so such sizes are refused on the host.
  const long ent = (long)e * a.P * a.K;
  const int total = a.P * a.K;
  for (int q = tid; q < a.groups; q += kLT) bucket[q] = 0;
  __syncthreads();
  constexpr int kBatch = 8;   // terms a thread reads at once
  for (int q0 = tid; q0 < total; q0 += kLT * kBatch) {
    unsigned v[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) v[u] = q0 + u * kLT < total ? a.idx[ent + q0 + u * kLT] : -1;
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (v[u] < (unsigned)a.Q) atomicAdd(&bucket[v[u] / 64], 1);
  }
  __syncthreads();
  int carry = 0;
  for (int q0 = 0; q0 < a.groups; q0 += kLT) {
    const int q = q0 + tid, n = q < a.groups ? bucket[q] : 0;
    int s = n;
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(s, o, 64);
      if ((tid & 63) >= o) s += u;
    }
    __syncthreads();
    if ((tid & 63) == 63) cnt[wave] = s;
    __syncthreads();
    int all = 0;
    for (int w = 0; w < kLT / 64; ++w) {
      if (w < wave) s += cnt[w];
      all += cnt[w];
    }
    if (q < a.groups) {
      bucket[q] = carry + s - n;
      a.first_rec[(long)e * (a.groups + 1) + q] = carry + s - n;
    }
    carry += all;
  }
  if (tid == 0) a.first_rec[(long)e * (a.groups + 1) + a.groups] = carry;
  __syncthreads();
  for (int q0 = tid; q0 < total; q0 += kLT * kBatch) {
    unsigned v[kBatch];
    int p[kBatch];
    float pi[kBatch], l[kBatch], g[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int q = q0 + u * kLT;
      const bool in = q < total;
      p[u] = in ? q / a.K : 0;
      v[u] = in ? a.idx[ent + q] : -1;
      pi[u] = in && a.prob ? a.prob[ent + q] : 1.f;
      l[u] = a.lse[(long)e * a.P + p[u]];
      g[u] = a.g[(long)e * a.P + p[u]];
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (v[u] < (unsigned)a.Q) {
        const int at = atomicAdd(&bucket[v[u] / 64], 1);
        const bool out = fabsf(l[u]) == INFINITY || pi[u] == 0.f;
        a.rec[ent + at] = make_uint2((unsigned)p[u] << 6 | (v[u] & 63), __float_as_uint(out ? 0.f : g[u] * pi[u]));
      }
  }
  if (!a.shared) return;
  const int i = a.e1[e], j = a.e2[e];
  int rank = 0;
  for (int q = tid; q < e; q += kLT) rank += a.e1[q] == i && a.e2[q] == j;
  for (int o = 32; o; o >>= 1) rank += __shfl_xor(rank, o, 64);
  __syncthreads();
  if ((tid & 63) == 0) cnt[wave] = rank;
  __syncthreads();
  rank = 0;
  for (int w = 0; w < kLT / 64; ++w) rank += cnt[w];
  for (int q0 = 0; q0 < a.E; q0 += kLT) {
    const int q = q0 + tid;
    const bool rev = q < a.E && a.e1[q] == j && a.e2[q] == i;
    const unsigned long long bal = __ballot(rev);
    __syncthreads();
    if ((tid & 63) == 0) cnt[wave] = __popcll(bal);
    __syncthreads();
    int at = __popcll(bal & ((1ull << (tid & 63)) - 1));
    for (int u = 0; u < wave; ++u) at += cnt[u];
    if (rev && at == rank) a.partner[e] = q;
    for (int w = 0; w < kLT / 64; ++w) rank -= cnt[w];
    if (rank < 0) break;
  }
}

// Whether edge e takes part: both ends are frames and a row has a target.
__device__ __forceinline__ bool edge_in(const BwdArgs& a, int e) {
  return (unsigned)a.e1[e] < (unsigned)a.N1 && (unsigned)a.e2[e] < (unsigned)a.N2 && a.gmax[e] >= 0.f;
}
// The span of the row sums of two edges (empty where an edge has none that counts).
__device__ __forceinline__ float2 edge_range(const BwdArgs& a, int e, int r) {
  return make_float2(fminf(a.range[e].x, a.range[r].x), fmaxf(a.range[e].y, a.range[r].y));
}
// Whether it is done together with its reverse: the weights of both then come from
// one exponential (bwd_edge), which holds while their lse lie within 2^kRange.
__device__ __forceinline__ bool edge_paired(const BwdArgs& a, int e) {
  const int r = a.partner[e];
  if (r < 0 || !(a.gmax[r] >= 0.f) || ((a.flags[e] | a.flags[r]) & 2)) return false;
  const float2 span = edge_range(a, e, r);
  return span.x <= span.y && span.y - span.x <= kRange;
}

// One workgroup: the units of every frame slot's items and their running sum.
__global__ void __launch_bounds__(1024) corr_plan_kernel(BwdArgs a) {
  constexpr int kChunk = 1024;
  __shared__ int both[kChunk], src[kChunk], dst[kChunk];
  __shared__ float gm[kChunk];
  __shared__ long long wsum[16];
  const int tid = threadIdx.x;
  long long base = 0;
  for (int v0 = 0; v0 < a.V; v0 += kChunk) {
    both[tid] = src[tid] = dst[tid] = 0;
    gm[tid] = 0.f;
    __syncthreads();
    for (int e = tid; e < a.E; e += kChunk) {
      if (!edge_in(a, e)) continue;
      // the edge's slot as source, and as target (one tensor: both in f1's slots)
      const int vs = a.n1 ? a.e1[e] - v0 : -1;
      const int vd = a.shared ? a.e2[e] - v0 : a.V > a.n1 ? a.n1 + a.e2[e] - v0 : -1;
      const bool paired = edge_paired(a, e);
      if ((unsigned)vs < (unsigned)kChunk) {
        atomicAdd(paired ? &both[vs] : &src[vs], 1);
        atomicMax(reinterpret_cast<int*>(&gm[vs]), __float_as_int(a.gmax[e]));   // >= 0: ordered as integers
      }
      if ((unsigned)vd < (unsigned)kChunk) {
        if (!paired) atomicAdd(&dst[vd], 1);   // paired: its reverse counts it
        atomicMax(reinterpret_cast<int*>(&gm[vd]), __float_as_int(a.gmax[e]));
      }
    }
    __syncthreads();
    const int v = v0 + tid;
    long long u = 0;
    if (v < a.V) {
      const bool first = v < a.n1;
      const int tiles = first ? a.tiles1 : a.tiles2;
      u = (long long)tiles * ((both[tid] * (long long)kUnitBoth + src[tid] * (long long)kUnitSrc) * (y_tiles(a.Q) + 1) +
                              dst[tid] * (long long)kUnitDst * (y_tiles(a.P) + 1));
      a.expo[v] = g_exponent(gm[tid]);
    }
    // inclusive scan over the chunk
    long long s = u;
    for (int o = 1; o < 64; o <<= 1) {
      const long long w = __shfl_up(s, o, 64);
      if ((tid & 63) >= o) s += w;
    }
    if ((tid & 63) == 63) wsum[tid >> 6] = s;
    __syncthreads();
    for (int w = 0; w < (tid >> 6); ++w) s += wsum[w];
    if (v < a.V) a.first[v + 1] = base + s;
    if (v == 0) a.first[0] = 0;
    long long all = 0;
    for (int w = 0; w < 16; ++w) all += wsum[w];
    base += all;
    __syncthreads();
  }
}

// Units of one workgroup's share.
__device__ __forceinline__ long long share_units(const BwdArgs& a) {
  return max((a.first[a.V] + a.G - 1) / a.G, (long long)kMinUnits);
}
// The frame slot that holds unit u (first[v] <= u < first[v + 1]).
__device__ __forceinline__ int slot_of(const BwdArgs& a, long long u) {
  int lo = 0, hi = a.V - 1;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (a.first[mid + 1] > u) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

constexpr int kHalves = 256;   // half tiles of one pass over an edge (longer frames: several passes)

// What a workgroup of the gradient kernel keeps in LDS.
template <int DP>
struct BwdShared {
  static constexpr int records = DP <= 128 ? 2048 : 512;   // sparse terms of a wave and a pass
  char tile[3][kRowsY * 2 * DP];           // rows aligned to their size; two tiles ahead
  float delta[4][32][32 * kXH<DP>];        // a wave's sparse terms of half a tile; zero between uses
  float expn[4][kRowsY], yg[4][kRowsY];    // the streamed queries' exponents and g, three tiles ahead
  float xg[bwd_rows(DP)];                  // the stationary queries' g
  int elist[kLT];
  int ecount[4];
  int ends[4][kHalves + 1];                // a wave's records: where those of each half tile end
  float val[4][records];                   // g pi
  unsigned short pos[4][records];          // y << 6 | x in the half tile
};

// The steps [t0, t1) of one edge (es: x are its queries) and / or its reverse
// (ed: the streamed rows y are its queries; NEG: some g of it are negative, which
// the exponents do not hold).
//
// The sparse targets (g pi at (y, x)) go through a dense, wave-private LDS image
// of half a tile, used only where there is one: the subtraction happens in fp32,
// before the rounding (p - pi of a well-trained row is a small difference).
// Before the steps a wave sorts the terms of its rows (its own targets, and the
// edge kernel's records of its keys) by half tile into LDS; where they do not fit,
// it reads them again at each half tile that has some.
template <typename T, int DP, bool SRC, bool DST, bool NEG>
__device__ __forceinline__ void bwd_edge(const BwdArgs& a, BwdShared<DP>& sh, int es, int ed, int t0, int t1, int R,
                                         int x0, int ex, const typename Op<T>::vec8 (&b)[kXH<DP>][DP / 16],
                                         floatx16 (&acc)[kXH<DP>][DP / 32]) {
  typedef typename Op<T>::vec8 vec8;
  typedef const __attribute__((address_space(3))) vec8* ptr;
  constexpr int RB = 2 * DP, KD = DP / 16, XH = kXH<DP>, XW = 32 * XH;   // XW rows a wave
  constexpr bool kScaled = !__is_same(T, __bf16);
  const int tid = fresh(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int n_y = SRC ? a.Q : a.P, K = a.K;
  const T* const frame = static_cast<const T*>(SRC ? a.f2 : a.f1) + (long)(SRC ? a.e2[es] : a.e1[ed]) * n_y * a.D;
  const float mul = ldexpf(1.f, ex), fex = (float)ex;
  float lx[XH], gx[XH], ax[XH];
  bool live = false;   // a stationary row has a target
  constexpr int kBatch = 8;   // sparse terms a lane reads at once
  // Both directions: with m the middle of the row sums, g1 p1 + g2 p2 = u (2^b g1 + A B)
  // where u = 2^(c s - lse_x - b), A = 2^(lse_x - m + b), B = 2^(v_y + m): one exponential
  // a pair of rows. b = kRange / 2, and lse_x := m in a left-out row x: then u <= 1
  // wherever x or y has a target, and is clamped to that where neither has, so that
  // it stays finite there and the factor 0 holds. u underflows where
  // c s < lse_x + b - 126: there p2 = 2^(c s - lse_y), with lse_x - lse_y up to kRange,
  // is below 2^(1.5 kRange - 126) = 2^-66.
  float mid = 0.f;
  if constexpr (SRC && DST) {
    const float2 span = edge_range(a, es, ed);
    mid = 0.5f * (span.x + span.y);
  }
  if constexpr (SRC) {
    bool any = false;
#pragma unroll
    for (int j = 0; j < XH; ++j) {
      const int x = x0 + wave * XW + 32 * j + (lane & 31);
      lx[j] = x < R ? a.lse[(long)es * a.P + x] : INFINITY;
      if (fabsf(lx[j]) == INFINITY) lx[j] = INFINITY;
      gx[j] = lx[j] == INFINITY ? 0.f : lx[j] == lx[j] ? a.g[(long)es * a.P + x] * mul : NAN;
      any |= lx[j] != INFINITY;
      if constexpr (SRC && DST) {
        if (lx[j] == INFINITY) lx[j] = mid;
        ax[j] = __builtin_amdgcn_exp2f(lx[j] - mid + 0.5f * kRange);
        lx[j] += 0.5f * kRange;
      }
      if (h == 0) sh.xg[wave * XW + 32 * j + lane] = gx[j];
      if constexpr (SRC && DST) gx[j] *= __builtin_amdgcn_exp2f(0.5f * kRange);
    }
    live = __syncthreads_or(any);
    if (!DST && !live) return;   // every row left out: nothing here, whatever the keys hold
  }
  // f(y, x, value) for the sparse terms of the streamed rows [ya, yb) and the wave's
  // rows x (from 0), over its lanes
  auto each_term = [&](int ya, int yb, auto f) {
    const int v = fresh(lane);
    if constexpr (SRC) {
      const long first = (long)es * a.P + x0 + wave * XW;
      const int n = min(XW, R - x0 - wave * XW) * K;
      const float inv = 1.f / (float)K;   // q / K by a product: q < 2^12, its distance from a whole number 2^-7
#pragma unroll 1
      for (int q0 = 0; q0 < n; q0 += 64 * kBatch) {
        int y[kBatch];
        float pi[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int q = q0 + 64 * u + v;
          y[u] = q < n ? a.idx[first * K + q] : -1;
          pi[u] = q < n && a.prob ? a.prob[first * K + q] : 1.f;
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          if (q0 + 64 * u >= n) break;
          if (y[u] >= ya && y[u] < yb && pi[u] != 0.f) {
            const int r = (int)(((float)(q0 + 64 * u + v) + 0.5f) * inv);
            f(y[u], r, sh.xg[wave * XW + r] * pi[u]);
          }
        }
      }
    }
    if constexpr (DST) {
      // the wave's rows are one group of 64 keys, or half of one
      const int x = x0 + wave * XW, group = x / 64;
      if (x < R) {
        const int* p = a.first_rec + (long)ed * (a.groups + 1) + group;
        const int lo = __builtin_amdgcn_readfirstlane(p[0]), hi = __builtin_amdgcn_readfirstlane(p[1]);
        const uint2* rec = a.rec + (long)ed * a.P * K;
#pragma unroll 1
        for (int q0 = lo; q0 < hi; q0 += 64 * kBatch) {
          uint2 r[kBatch];
#pragma unroll
          for (int u = 0; u < kBatch; ++u)
            r[u] = q0 + 64 * u + v < hi ? rec[q0 + 64 * u + v] : make_uint2(0xffffffffu, 0u);
#pragma unroll
          for (int u = 0; u < kBatch; ++u) {
            if (q0 + 64 * u >= hi) break;
            const int y = r[u].x >> 6, k = (int)(r[u].x & 63) - (x & 63);
            if (y >= ya && y < yb && (XW == 64 || (k >= 0 && k < XW))) f(y, k, __uint_as_float(r[u].y) * mul);
          }
        }
      }
    }
  };
  bool stored;
  {
    // count by half tile, running sum, place: all of it the wave's own
    int (&ends)[kHalves + 1] = sh.ends[wave];
    const int ya = t0 * kRowsY, yb = t1 * kRowsY;
    for (int q = lane; q <= kHalves; q += 64) ends[q] = 0;
    each_term(ya, yb, [&](int y, int, float) { atomicAdd(&ends[(y - ya) / 32], 1); });
    int carry = 0;
#pragma unroll 1
    for (int q = lane; q < kHalves; q += 64) {
      const int n = ends[q];
      int s = n;
      for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(s, o, 64);
        if (lane >= o) s += u;
      }
      ends[q] = carry + s - n;
      carry += __shfl(s, 63, 64);
    }
    stored = carry <= BwdShared<DP>::records;
    if (stored)
      each_term(ya, yb, [&](int y, int x, float value) {
        const int at = atomicAdd(&ends[(y - ya) / 32], 1);   // ends as the half tile's end
        sh.pos[wave][at] = (unsigned short)((y & 31) << 6 | x);
        sh.val[wave][at] = value;
      });
    else   // the starts become ends
      for (int q = lane; q < kHalves; q += 64) ends[q] = q + 1 < kHalves ? ends[q + 1] : carry;
  }
  // Streamed queries: |g| mul p2 = 2^(c s + v + ex) with their exponents v.  They
  // are staged a tile further ahead: v = -inf marks a row without a gradient; where
  // such rows are not finite they are staged as zeros (unless they are live keys:
  // then the NaN is theirs).
  const rsrc_t rex = make_rsrc(a.expn + (long)ed * y_tiles(a.P) * kRowsY, (unsigned)y_tiles(a.P) * kRowsY * 4);
  const rsrc_t rg = make_rsrc(a.g + (long)ed * a.P, (unsigned)a.P * 4);
  auto stage_rows = [&](int t) {
    if (DST && wave == 0) dma4(rex, lds_addr(sh.expn[(t - t0) & 3]), (unsigned)(t * kRowsY + lane) * 4);
    if (DST && wave == 1) dma4(rg, lds_addr(sh.yg[(t - t0) & 3]), (unsigned)(t * kRowsY + lane) * 4);
  };
  const int ef = DST ? a.flags[ed] : 0;
  const bool holes = (ef & 1) && !(SRC && live);
  unsigned off[kDmas<DP>];
  lane_offsets<DP>(off, a.D, wave, lane);
  auto stage = [&](int t, int buf) {
    if (!holes)
      stage_tile<T, DP>(frame, sh.tile[buf], t * kRowsY, n_y, a.D, off, wave, lane, [](int) { return false; });
    else
      stage_tile<T, DP>(frame, sh.tile[buf], t * kRowsY, n_y, a.D, off, wave, lane,
                        [&](int row) { return sh.expn[(t - t0) & 3][row] == -INFINITY; });
  };
  // Before the loop: the row data of three tiles, the features of two.
  stage_rows(t0);
  if (t0 + 1 < t1) stage_rows(t0 + 1);
  if (t0 + 2 < t1) stage_rows(t0 + 2);
  if (holes) {
    loads_done();
    __syncthreads();
  }
  stage(t0, 0);
  if (t0 + 1 < t1) stage(t0 + 1, 1);
  loads_done();
  __syncthreads();
  // Both directions: the exponents v become B in place, a step before their tile's, by
  // one wave for all (each lane for itself: 32 exponentials a step).
  auto make_b = [&](int t) {
    float& v = sh.expn[(t - t0) & 3][lane];
    v = __builtin_amdgcn_exp2f(v + (mid + fex));
  };
  if constexpr (SRC && DST) {
    if (wave == 3) make_b(t0);
    __syncthreads();
  }
  int buf = 0;   // of tile t
  // Half 1's second product of a tile is done in the next step, while that one's
  // operands are on their way (nothing yet: zeros), where there are registers to
  // keep its operands (D <= 128).
  constexpr bool kDefer = DP <= 128;
  constexpr int kS = KD * XH, kP = 2 * (DP / 32) * XH;   // matrix instructions of a half's logits, second product
  vec8 ds[XH][2], ft[2][2][DP / 32];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int j = 0; j < XH; ++j) ds[j][k] = vec8{};
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) ft[1][k][d] = vec8{};
  }
  auto product = [&](int half, int n) {
    const int k = n / (kP / 2), d = n % (kP / 2) / XH, j = n % XH;
    acc[j][d] = Op<T>::mfma(ft[half][k][d], ds[j][k], acc[j][d]);
  };
  for (int t = t0; t < t1; ++t) {
    const int ahead = buf == 0 ? 2 : buf - 1;
    const unsigned cur = lds_addr(sh.tile[buf]), row0 = row_addr<DP>(cur, fresh(lane));
    vec8 fa[2][KD];
    auto read_row = [&](int n) {   // the n-th of the 2 KD operands of the logits
      const int k = n / KD, d = n % KD;
      fa[k][d] = *(ptr)(uintptr_t)((row0 ^ (d << 5)) + k * 64 * DP);
    };
    // The second product's operand: rows d of the transposed tile.  As the address
    // lane 4 q + p of its 16-lane group a lane points at row 16 k + 8 u + 4 h + q,
    // values 32 d + 16 ((lane >> 4) & 1) + 4 p .. + 3; d and u move the swizzled
    // address by an XOR, k and u by whole rows.
    const int tv = fresh(lane), q4 = ((tv & 15) >> 2) + 4 * (tv >> 5), s0 = 2 * ((tv >> 4) & 1) + ((tv >> 1) & 1);
    const unsigned tr0 = cur + q4 * RB + ((s0 ^ swz<DP>(q4)) << 4) + (tv & 1) * 8;
    auto transposed = [&](int d, int k) {
      struct { short4_t lo, hi; } both = {
          __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) short4_t*)(uintptr_t)((tr0 ^ (d << 6)) + 16 * k * RB)),
          __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) short4_t*)(uintptr_t)((tr0 ^ (d << 6 | 32)) + (16 * k + 8) * RB))};
      return __builtin_bit_cast(vec8, both);
    };
    floatx16 sc[2][XH];
    float wg[XH][16];
    auto logit = [&](int k, int n) {
      sc[k][n % XH] = Op<T>::mfma(fa[k][n / XH], b[n % XH][n / XH], sc[k][n % XH]);
    };
    auto zero = [&](int k) {
#pragma unroll
      for (int j = 0; j < XH; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[k][j][i] = 0.f;
    };
    float ve[16];   // the exponents (both directions: B) of the half's rows in this lane's places
    auto exponents = [&](int k) {
      if constexpr (DST)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float4 v = *reinterpret_cast<const float4*>(&sh.expn[(t - t0) & 3][32 * k + 8 * q + 4 * h]);
          const float vq[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int u = 0; u < 4; ++u)
            ve[4 * q + u] = !SRC && kScaled ? vq[u] + fex : vq[u];
        }
    };
    // The weights of half k with N matrix instructions between them, in exactly this
    // order (left to itself the scheduler puts them one after the other): per matrix
    // instruction the exponentials of some elements and the sums of the ones before.
    auto weights = [&](int k, auto matrix, auto n_tag) {
      constexpr int N = decltype(n_tag)::value, E = 16 * XH / N;   // elements per matrix instruction
      static_assert(16 * XH % N == 0, "elements per matrix instruction");
      float p1[2][E];
      auto finish = [&](int n) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int j = (n * E + e) / 16, q = (n * E + e) % 16;
          if constexpr (SRC) wg[j][q] = p1[n & 1][e] * (DST ? fmaf(ax[j], ve[q], gx[j]) : gx[j]);
        }
      };
#pragma unroll
      for (int n = 0; n < N; ++n) {
        matrix(n);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int j = (n * E + e) / 16, q = (n * E + e) % 16;
          if constexpr (!SRC) {
            wg[j][q] = __builtin_amdgcn_exp2f(fmaf(sc[k][j][q], a.c, ve[q]));
            if constexpr (NEG)
              if (sh.yg[(t - t0) & 3][32 * k + 8 * (q >> 2) + 4 * h + (q & 3)] < 0.f) wg[j][q] = -wg[j][q];
          } else {
            const float u = __builtin_amdgcn_exp2f(fmaf(sc[k][j][q], a.c, -lx[j]));
            // (the clamp takes a NaN logit, of a left-out row, to 0)
            p1[n & 1][e] = __builtin_amdgcn_fmed3f(u, 0.f, 1.f);
          }
        }
        if (n) finish(n - 1);
        __builtin_amdgcn_sched_barrier(0);
      }
      finish(N - 1);
    };
    // the wave's records of this tile: [lo, mid) in half 0, [mid, hi) in half 1
    const int half = 2 * (t - t0), br[3] = {half ? sh.ends[wave][half - 1] : 0, sh.ends[wave][half], sh.ends[wave][half + 1]};
    auto sparse_and_round = [&](int k) {
      const int lo = __builtin_amdgcn_readfirstlane(br[k]), hi = __builtin_amdgcn_readfirstlane(br[k + 1]);
      if (lo < hi) {
        float (&dl)[32][XW] = sh.delta[wave];
        const int v = fresh(lane), ya = t * kRowsY + 32 * k;
        if (stored)
          for (int q = lo + v; q < hi; q += 64) atomicAdd(&dl[0][0] + (XW == 64 ? sh.pos[wave][q] : (sh.pos[wave][q] >> 6) * XW + (sh.pos[wave][q] & 63)), sh.val[wave][q]);
        else
          each_term(ya, ya + 32, [&](int y, int x, float value) { atomicAdd(&dl[y - ya][x], value); });
        const float* col = &dl[4 * (v >> 5)][v & 31];
#pragma unroll
        for (int j = 0; j < XH; ++j)
#pragma unroll
          for (int q = 0; q < 16; ++q) wg[j][q] -= col[(8 * (q >> 2) + (q & 3)) * XW + 32 * j];
        if (stored)
          for (int q = lo + v; q < hi; q += 64) (&dl[0][0])[XW == 64 ? sh.pos[wave][q] : (sh.pos[wave][q] >> 6) * XW + (sh.pos[wave][q] & 63)] = 0.f;
        else
          for (int q = v; q < 32 * XW / 4; q += 64) reinterpret_cast<float4*>(&dl[0][0])[q] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int j = 0; j < XH; ++j)
#pragma unroll
        for (int q = 0; q < 16; ++q) ds[j][q >> 3][q & 7] = (T)wg[j][q];
      if (lo < hi) {   // what the rounding left
#pragma unroll
        for (int j = 0; j < XH; ++j)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            vec8 high = ds[j][u], low;
            asm("" : "+v"(high));   // (or every step converts one value at a time, for these)
#pragma unroll
            for (int q = 0; q < 8; ++q) low[q] = (T)(wg[j][8 * u + q] - (float)high[q]);
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) acc[j][d] = Op<T>::mfma(ft[k][u][d], low, acc[j][d]);
          }
      }
    };
    auto read_transposed = [&](int half, int n) {   // the n-th of DP / 16
      const int k = n / (DP / 32), d = n % (DP / 32);
      ft[half][k][d] = transposed(d, 2 * half + k);
    };
    // A step: the last half's second product, half 0's logits; half 1's logits between
    // half 0's weights; half 0's second product between half 1's weights.  The reads
    // of shared memory, which take the four waves of a workgroup about 1100 clocks a step,
    // stand between the matrix instructions too.
    zero(0);
    zero(1);
    if constexpr (kDefer) {
#pragma unroll
      for (int n = 0; n < kP; ++n) {
        product(1, n);
#pragma unroll
        for (int q = 2 * KD * n / kP; q < 2 * KD * (n + 1) / kP; ++q) read_row(q);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int q = 0; q < 2 * KD; ++q) read_row(q);
    }
    if (t + 2 < t1) {
      if (t + 3 < t1) stage_rows(t + 3);   // before the tile: landed when this step ends
      stage(t + 2, ahead);
    }
    if constexpr (SRC && DST) {
      if (wave == 3 && t + 1 < t1) make_b(t + 1);
    }
    exponents(0);
#pragma unroll
    for (int n = 0; n < kS; ++n) {
      logit(0, n);
#pragma unroll
      for (int q = KD * n / kS; q < KD * (n + 1) / kS; ++q) read_transposed(0, q);
      __builtin_amdgcn_sched_barrier(0);
    }
    weights(0, [&](int n) { logit(1, n); }, std::integral_constant<int, kS>());
    exponents(1);
    sparse_and_round(0);
    __builtin_amdgcn_sched_barrier(0);
    weights(1, [&](int n) {
      product(0, n);
#pragma unroll
      for (int q = KD * n / kP; q < KD * (n + 1) / kP; ++q) read_transposed(1, q);
    }, std::integral_constant<int, kP>());
    sparse_and_round(1);
    if constexpr (!kDefer) {
#pragma unroll
      for (int n = 0; n < kP; ++n) product(1, n);
    }
    buf = buf == 2 ? 0 : buf + 1;
    // tile t + 1 and t + 3's row data, which the next step's stage reads, have landed;
    // the loads of tile t + 2 stay in flight
    if (t + 3 < t1) loads_left<kDmas<DP>>();
    else loads_done();
    __syncthreads();
  }
  if constexpr (kDefer) {
#pragma unroll
    for (int n = 0; n < kP; ++n) product(1, n);
  }
}

// The edges of one kind at frame n, 256 at a time, in order; `at`: units of the
// item before this kind's first edge (moved past its last), [u0, u1) the units
// that are done here.
template <typename T, int DP, bool SRC, bool DST, bool NEG = false>
__device__ __forceinline__ void bwd_kind(const BwdArgs& a, BwdShared<DP>& sh, int n, long long& at, long long u0,
                                         long long u1, int R, int x0, int ex,
                                         const typename Op<T>::vec8 (&b)[kXH<DP>][DP / 16],
                                         floatx16 (&acc)[kXH<DP>][DP / 32]) {
  const int tid = fresh(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  constexpr int unit = SRC && DST ? kUnitBoth : SRC ? kUnitSrc : kUnitDst;
  const int nt = y_tiles(SRC ? a.Q : a.P);
  for (int e0 = 0; e0 < a.E && at < u1; e0 += kLT) {
    const int e = e0 + tid;
    bool in = e < a.E && (SRC ? a.e1 : a.e2)[e] == n;
    if (in) in = edge_in(a, e) && (SRC && DST) == edge_paired(a, e) && (SRC || ((a.flags[e] & 2) != 0) == NEG);
    const unsigned long long bal = __ballot(in);
    if (lane == 0) sh.ecount[wave] = __popcll(bal);
    __syncthreads();
    int pos = __popcll(bal & ((1ull << lane) - 1));
    for (int q = 0; q < wave; ++q) pos += sh.ecount[q];
    if (in) sh.elist[pos] = e;
    const int cnt = __builtin_amdgcn_readfirstlane(sh.ecount[0] + sh.ecount[1] + sh.ecount[2] + sh.ecount[3]);
    __syncthreads();
    for (int q = 0; q < cnt && at < u1; ++q, at += (long long)(nt + 1) * unit) {   // one step's time to begin an edge
      // a step is done by the share that its first unit lies in
      const int t0 = (int)max(0ll, (u0 - at + unit - 1) / unit), t1 = (int)min((long long)nt, (u1 - at + unit - 1) / unit);
      if (t0 >= t1) continue;
      const int eq = __builtin_amdgcn_readfirstlane(sh.elist[q]);
      const int er = SRC && DST ? __builtin_amdgcn_readfirstlane(a.partner[eq]) : eq;
      for (int t = t0; t < t1; t += kHalves / 2)
        bwd_edge<T, DP, SRC, DST, NEG>(a, sh, eq, er, t, min(t1, t + kHalves / 2), R, x0, ex, b, acc);
    }
    __syncthreads();
  }
}

// One workgroup: its share of the units, item by item.
template <typename T, int DP>
__global__ void __launch_bounds__(kLT, 1) corr_loss_bwd_kernel(BwdArgs a) {
  constexpr bool kScaled = !__is_same(T, __bf16);
  constexpr int XH = kXH<DP>, rows = bwd_rows(DP);
  __shared__ __attribute__((aligned(1024))) BwdShared<DP> sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
  const int block = xcd_item(blockIdx.x, a.G);
  if (block >= a.G) return;
  const long long share = share_units(a), all = a.first[a.V];
  long long u = block * share;
  const long long end = min(u + share, all);
  for (int q = lane; q < 32 * 32 * XH; q += 64) (&sh.delta[wave][0][0])[q] = 0.f;
  while (u < end) {
    const int v = slot_of(a, u);
    const bool second = v >= a.n1;
    const int n = second ? v - a.n1 : v, tiles = second ? a.tiles2 : a.tiles1, R = second ? a.Q : a.P;
    const long long per = (a.first[v + 1] - a.first[v]) / tiles;   // units of each of the frame's items
    const int w = (int)((u - a.first[v]) / per), x0 = w * rows;
    const long long item = a.first[v] + w * per;
    const long long u0 = u - item, u1 = min(per, end - item);
    typename Op<T>::vec8 b[XH][DP / 16];
    floatx16 acc[XH][DP / 32];
#pragma unroll
    for (int j = 0; j < XH; ++j) {
      load_rows<T, DP>(b[j], static_cast<const T*>(second ? a.f2 : a.f1) + (long)n * R * a.D,
                       x0 + (wave * XH + j) * 32 + (lane & 31), R, a.D, h);
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int q = 0; q < 16; ++q) acc[j][d][q] = 0.f;
    }
    const int ex = kScaled ? a.expo[v] : 0;
    // the kinds one after the other: in one loop the compiler keeps the values of
    // all of them in registers and spills
    long long at = 0;
    if (a.shared) bwd_kind<T, DP, true, true>(a, sh, n, at, u0, u1, R, x0, ex, b, acc);
    if (!second) bwd_kind<T, DP, true, false>(a, sh, n, at, u0, u1, R, x0, ex, b, acc);
    if (second || a.shared) {
      bwd_kind<T, DP, false, true>(a, sh, n, at, u0, u1, R, x0, ex, b, acc);
      bwd_kind<T, DP, false, true, true>(a, sh, n, at, u0, u1, R, x0, ex, b, acc);
    }

    const float out = a.out_scale * (kScaled ? ldexpf(1.f, -ex) : 1.f);
    const bool whole = u0 == 0 && u1 == per;
#pragma unroll
    for (int j = 0; j < XH; ++j) {
      const int x = x0 + (wave * XH + j) * 32 + (fresh(lane) & 31);
      if (x >= R) continue;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = 32 * d + 8 * q + 4 * h;
          if (c >= a.D) continue;
          float o[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) o[k] = acc[j][d][4 * q + k] * out;
          if (whole) {
            typedef T t4 __attribute__((ext_vector_type(4)));
            *reinterpret_cast<t4*>(static_cast<T*>(second ? a.d2 : a.d1) + ((long)n * R + x) * a.D + c) =
                t4{(T)o[0], (T)o[1], (T)o[2], (T)o[3]};
          } else {
            float* p = a.part + ((long)(2 * block + (u0 == 0)) * rows + (x - x0)) * a.D + c;
            *reinterpret_cast<float4*>(p) = make_float4(o[0], o[1], o[2], o[3]);
          }
        }
    }
    u = item + u1;
  }
}

// kJoin workgroups an item: add up, in order, the parts of one that several
// shares have worked on; zeros where no edge reaches the frame.
template <typename T>
__global__ void __launch_bounds__(kLT) corr_loss_join_kernel(BwdArgs a) {
  const int items1 = a.n1 * a.tiles1;
  const bool second = (int)blockIdx.x >= items1;
  const int w = second ? blockIdx.x - items1 : blockIdx.x, tiles = second ? a.tiles2 : a.tiles1;
  const int n = w / tiles, rows = bwd_rows(a.D), x0 = w % tiles * rows, R = second ? a.Q : a.P, v = second ? a.n1 + n : n;
  const long long per = (a.first[v + 1] - a.first[v]) / tiles, item = a.first[v] + w % tiles * per;
  const long long share = share_units(a);
  const int b0 = (int)(item / share), b1 = per ? (int)((item + per - 1) / share) : b0;
  if (per && b0 == b1) return;
  T* d = static_cast<T*>(second ? a.d2 : a.d1) + ((long)n * R + x0) * a.D;
  const int total = min(rows, R - x0) * a.D;
  for (int q = (blockIdx.y * kLT + threadIdx.x) * 4; q < total; q += kLT * 4 * kJoin) {
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (per)
#pragma unroll 4
      for (int b = b0; b <= b1; ++b) {
        const float4 p = *reinterpret_cast<const float4*>(a.part + (long)(2 * b + (b == b0)) * rows * a.D + q);
        s.x += p.x;
        s.y += p.y;
        s.z += p.z;
        s.w += p.w;
      }
    typedef T t4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<t4*>(d + q) = t4{(T)s.x, (T)s.y, (T)s.z, (T)s.w};
  }
}

// Shares of the keys: the split with the least steps of a workgroup one after the
// other, a share costing about two steps more than its tiles (its start and join).
int fwd_split(int E, int P, int Q, int D) {
  const long blocks = (long)E * ceil_div(P, fwd_rows(D)), tiles = ceil_div(Q, kRowsY);
  const long at_once = (long)fwd_groups(D) * device_cu_count();
  long best = 1, least = -1;
  const long most = std::min<long>(tiles, std::max<long>(8, at_once / std::max<long>(1, blocks)));
  for (long s = 1; s <= most; s += 1 + s / 64) {
    const long steps = (blocks * s + at_once - 1) / at_once * ((tiles + s - 1) / s + 2);
    if (least < 0 || steps < least) best = s, least = steps;
  }
  return (int)best;
}

// Workgroups of the gradient kernel: as many as run at once, one a CU by its registers.
int bwd_groups() { return device_cu_count(); }

// The gradient's workspace, in bytes from its start.
struct BwdSpace {
  size_t gmax, partner, flags, range, first, expo, first_rec, rec, expn, part, bytes;
};
BwdSpace bwd_space(int E, int P, int Q, int V, int D, int K) {
  auto up = [](size_t n) { return (n + 15) / 16 * 16; };
  BwdSpace s{};
  s.partner = s.gmax + up((size_t)E * 4);
  s.flags = s.partner + up((size_t)E * 4);
  s.range = s.flags + up((size_t)E * 4);
  s.first = s.range + up((size_t)E * 8);
  s.expo = s.first + up(((size_t)V + 1) * 8);
  s.first_rec = s.expo + up((size_t)V * 4);
  s.rec = s.first_rec + up((size_t)E * (ceil_div(Q, 64) + 1) * 4);
  s.expn = s.rec + up((size_t)E * P * K * 8);
  s.part = s.expn + (size_t)E * y_tiles(P) * kRowsY * 4;
  s.bytes = s.part + (size_t)2 * bwd_groups() * bwd_rows(D) * D * 4;
  return s;
}

int corr_loss_check(const std::string& w, int dtype, int E, int N1, int P, int N2, int Q, int D, int K, float scale,
                    float T) {
  if (dtype != 0 && dtype != 3) return fail(kInvalidArgument, w + ": features must be float16 or bfloat16");
  if (E < 0 || N1 < 0 || N2 < 0 || P < 0 || Q <= 0 || D <= 0 || D % 8 || D > 256 || K < 1 || K > kMaxK)
    return fail(kInvalidArgument, w + ": bad arguments (Q > 0, 0 < D <= 256, D % 8 == 0, 1 <= K <= 64)");
  if (!(scale > 0.f) || !std::isfinite(scale) || !(T > 0.f) || !std::isfinite(T))
    return fail(kInvalidArgument, w + ": scale and temperature must be positive and finite");
  // (a product of 0 times a key past the end's -inf, or an infinite one, would be NaN)
  for (const float f : {scale / T, scale / T * kLog2e, scale * T, T * T})
    if (!(f >= FLT_MIN && f <= FLT_MAX))
      return fail(kInvalidArgument, w + ": scale / temperature, their product and temperature^2 must be normal numbers");
  if (std::max(P, Q) > 64 * kMaxGroups || (long)std::max(P, Q) * D * 2 > 0x7fffffffL || (long)P * K > 0x1fffffffL || (long)E * std::max(1, ceil_div(P, kRowsB)) > 0x3fffffL ||
      (long)(N1 + (long)N2) * ceil_div(std::max(P, Q), kRowsB) > 0x3fffffL)
    return fail(kUnsupported, w + ": maps too large");
  return kOk;
}

bool unaligned(const void* p) { return reinterpret_cast<uintptr_t>(p) & 15; }

}  // namespace

}  // namespace droid

using namespace droid;

#define CORR_DIMS(T, LAUNCH) \
  if (D <= 64) { LAUNCH(T, 64); } else if (D <= 128) { LAUNCH(T, 128); } else { LAUNCH(T, 256); }
#define CORR_TYPES(LAUNCH) \
  if (dtype == 0) { CORR_DIMS(_Float16, LAUNCH) } else { CORR_DIMS(__bf16, LAUNCH) }

extern "C" {

size_t droid_corr_loss_workspace(int E, int N1, int P, int N2, int Q, int D, int K, int backward) {
  if (E <= 0 || N1 < 0 || P <= 0 || N2 < 0 || Q <= 0 || D <= 0 || K <= 0) return 0;
  if (!backward) return (size_t)E * P * fwd_split(E, P, Q, D) * sizeof(float2);
  return bwd_space(E, P, Q, N1 + N2, D, K).bytes;
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
  if (!ws || ws_bytes < droid_corr_loss_workspace(E, N1, P, N2, Q, D, K, 0))
    return fail(kInvalidArgument, what + ": workspace too small");
  FwdArgs a{fmap1, fmap2, f1, f2, idx, static_cast<float2*>(ws), E, N1, P, N2, Q, D, K, ceil_div(P, fwd_rows(D)),
            fwd_split(E, P, Q, D), 0, scale / temperature * kLog2e};
  a.items = E * a.tiles * a.S;
#define LSE(T, DP) corr_lse_kernel<T, DP><<<(a.items + 7) / 8 * 8, kLT, 0, stream>>>(a)
  CORR_TYPES(LSE)
#undef LSE
  DROID_LAUNCH_CHECK();
  RowArgs r{fmap1, fmap2, f1, f2, idx, logits, a.part, loss, lse, logits ? prob : nullptr, N1, P, N2, Q, D, K, a.S,
            (long)E * P, 1.f / temperature, temperature * temperature, a.c};
  const int grid = (int)((r.rows + kLT / 16 - 1) / (kLT / 16));
#define ROW(SLOTS, BATCH)                                                                       \
  if (dtype == 0) corr_loss_row_kernel<_Float16, SLOTS, BATCH><<<grid, kLT, 0, stream>>>(r);    \
  else corr_loss_row_kernel<__bf16, SLOTS, BATCH><<<grid, kLT, 0, stream>>>(r)
  if (K == 1) {
    ROW(1, 1);
  } else if (K <= 16) {
    ROW(1, 4);
  } else {
    ROW(4, 4);
  }
#undef ROW
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
  // the reverse of an edge is looked for, and a frame's edges gathered, in the whole list
  if (E > kMaxEdges) return fail(kUnsupported, what + ": more than 65536 edges");
  if (!fmap1 || !fmap2 || !f1 || !f2 || !idx || !lse || !gloss || (!dfmap1 && !dfmap2))
    return fail(kInvalidArgument, what + ": null tensor");
  if (!prob && K != 1) return fail(kInvalidArgument, what + ": one target a row without weights");
  if (shared && (fmap1 != fmap2 || N1 != N2 || P != Q || dfmap2))
    return fail(kInvalidArgument, what + ": one shared feature tensor has one gradient");
  if (unaligned(fmap1) || unaligned(fmap2)) return fail(kInvalidArgument, what + ": features must be 16-B aligned");
  // the gradients that are wanted; a shared tensor's rows are counted once
  const int n1 = dfmap1 ? N1 : 0, n2 = dfmap2 ? N2 : 0;
  if (!ws || ws_bytes < droid_corr_loss_workspace(E, n1, P, n2, Q, D, K, 1))
    return fail(kInvalidArgument, what + ": workspace too small");
  if (n1 + n2 == 0) return kOk;
  char* const w = static_cast<char*>(ws);
  const BwdSpace sp = bwd_space(E, P, Q, n1 + n2, D, K);
  BwdArgs a{};
  a.f1 = fmap1, a.f2 = fmap2, a.e1 = f1, a.e2 = f2, a.idx = idx, a.prob = prob, a.lse = lse, a.g = gloss;
  a.d1 = dfmap1, a.d2 = dfmap2;
  a.gmax = reinterpret_cast<float*>(w + sp.gmax), a.partner = reinterpret_cast<int*>(w + sp.partner);
  a.first = reinterpret_cast<long long*>(w + sp.first), a.expo = reinterpret_cast<int*>(w + sp.expo);
  a.part = reinterpret_cast<float*>(w + sp.part), a.flags = reinterpret_cast<int*>(w + sp.flags);
  a.expn = reinterpret_cast<float*>(w + sp.expn), a.first_rec = reinterpret_cast<int*>(w + sp.first_rec);
  a.rec = reinterpret_cast<uint2*>(w + sp.rec), a.groups = ceil_div(Q, 64);
  a.range = reinterpret_cast<float2*>(w + sp.range);
  a.E = E, a.N1 = N1, a.P = P, a.N2 = N2, a.Q = Q, a.D = D, a.K = K, a.shared = shared != 0;
  a.tiles1 = ceil_div(P, bwd_rows(D)), a.tiles2 = ceil_div(Q, bwd_rows(D));
  a.n1 = n1, a.V = n1 + n2, a.G = bwd_groups();
  a.c = scale / temperature * kLog2e, a.out_scale = scale * temperature;
  corr_edge_kernel<<<E, kET, 0, stream>>>(a);
  DROID_LAUNCH_CHECK();
  corr_plan_kernel<<<1, 1024, 0, stream>>>(a);
  DROID_LAUNCH_CHECK();
  const int grid = (a.G + 7) / 8 * 8;
#define BWD(T, DP) corr_loss_bwd_kernel<T, DP><<<grid, kLT, 0, stream>>>(a)
  CORR_TYPES(BWD)
#undef BWD
  DROID_LAUNCH_CHECK();
  const int items = n1 * a.tiles1 + n2 * a.tiles2;
  if (dtype == 0) corr_loss_join_kernel<_Float16><<<dim3(items, kJoin), kLT, 0, stream>>>(a);
  else corr_loss_join_kernel<__bf16><<<dim3(items, kJoin), kLT, 0, stream>>>(a);
  DROID_LAUNCH_CHECK();
  return kOk;
}

}  // extern "C"
