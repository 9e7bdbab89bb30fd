// Group normalisation with the activation and residual add around it
// (modules/extractor.py: GroupNorm of BasicEncoder(norm_fn='group') and its
// ResidualBlocks), channels last, forward and backward.
//
// x is (N, HW, C), C = G cpg channels in G groups; per image and group, over
// M = HW cpg values:
//   n   = (x - mean) rstd w_c + b_c,   rstd = 1 / sqrt(var + eps), biased var
//   mode 0 relu(n)   1 relu(res + relu(n))   2 relu(n + res)   3 n   4 silu(n)
// backward, with dn = dy times the activation's slope and dres = dy times the
// outer ReLU's:
//   dw_c = sum dn xhat,  db_c = sum dn,
//   dx   = rstd (w dn - (sum_g w dn) / M - xhat (sum_g w dn xhat) / M)
//
// Every pass is a stream over maps, bound by HBM (or, for one frame, by the two
// launches): forward reads x twice and writes y; backward's first pass reads x,
// dy (and res) and writes dres, its second reads x and dy (dres) and writes dx.
// 28 maps of 32 x 160 x 256 in bf16, relu(res + relu(n)): 16 + 37 us forward,
// 50 + 40 us backward, 5.6 TB/s over what the passes move (a large copy: 5.1; the
// second passes find part of it in the last-level cache); what the operator cannot
// do without is 115 us of that copy.
//
// Layout of the work.  An image is a flat run of HW C values, cut into pieces
// of V = 16 B.  Piece f starts at channel (V f) mod C, so with A threads, A a
// multiple of C / gcd(C, V), a thread that takes pieces t, t + A, t + 2A, ...
// meets the same V channels every time: its channel constants stay in
// registers, and any C (odd ones too) streams with 16-B loads; only the last
// HW C mod V values of an image are read one by one.
//
// Statistics: a thread sums its values in fp32 relative to the first one it
// met (no cancellation where the mean is far from zero) over at most kFlush
// pieces, then adds them to 64-bit sums; everything after that is 64-bit and
// added in a fixed order, so results do not depend on the schedule.  The
// backward pass's sums of dn and dn xhat likewise.  mean and
// rstd are kept in 64 bits for the backward pass: where a ReLU's argument is
// within rounding of zero its sign is decided in 64 bits, because one wrong
// sign moves a whole gradient, not its last bit.
#include "common.hpp"

#include <algorithm>

namespace droid {

namespace {

constexpr int kGnT = 512;      // threads; C / gcd(C, V) <= C <= kGnMaxC fits one thread per piece
constexpr int kGnMaxC = 512;
constexpr int kFlush = 32;     // pieces summed in fp32 before they go to 64 bits
constexpr float kTol = 1e-6f;  // 16 fp32 roundings: a ReLU argument below this share of its terms is re-done in 64 bits

enum { kRelu = 0, kResRelu = 1, kAddRelu = 2, kNone = 3, kSilu = 4 };

template <typename T>
struct Elem;
template <>
struct Elem<_Float16> {
  static constexpr int V = 8;
};
template <>
struct Elem<__bf16> {
  static constexpr int V = 8;
};
template <>
struct Elem<float> {
  static constexpr int V = 4;
};

template <typename T>
struct Piece {
  T v[Elem<T>::V];
};

// 16 B at any element's alignment (unaligned global accesses are legal)
template <typename T>
__device__ __forceinline__ Piece<T> load_piece(const T* p) {
  Piece<T> r;
  __builtin_memcpy(&r, p, 16);
  return r;
}
template <typename T>
__device__ __forceinline__ void store_piece(T* p, const Piece<T>& r) {
  __builtin_memcpy(p, &r, 16);
}
// the image's last, short piece: m values
template <typename T>
__device__ __forceinline__ Piece<T> load_tail(const T* p, int m) {
  Piece<T> r;
#pragma unroll
  for (int k = 0; k < Elem<T>::V; ++k) r.v[k] = k < m ? p[k] : (T)0.f;
  return r;
}
template <typename T>
__device__ __forceinline__ void store_tail(T* p, const Piece<T>& r, int m) {
#pragma unroll
  for (int k = 0; k < Elem<T>::V; ++k)
    if (k < m) p[k] = r.v[k];
}

__device__ __forceinline__ float param(const void* p, int dt, int c, float dflt) {
  if (!p) return dflt;
  if (dt == 1) return static_cast<const float*>(p)[c];
  if (dt == 0) return (float)static_cast<const _Float16*>(p)[c];
  return (float)static_cast<const __bf16*>(p)[c];
}

// The split of an image's pieces over threads and workgroups.
struct Split {
  long pieces;   // full pieces of one image
  int tail;      // values after them (< V)
  int active;    // threads that take pieces: a multiple of the channel pattern's period
  int blocks;    // workgroups an image: block s takes chunks (of `active` pieces) [chunks s / blocks, ...)
  long chunks;
};

inline int gcd_i(int a, int b) {
  while (b) {
    const int t = a % b;
    a = b;
    b = t;
  }
  return a;
}

inline Split gn_split(int N, int HW, int C, int V) {
  Split s;
  const long total = (long)HW * C;
  s.pieces = total / V;
  s.tail = (int)(total % V);
  const int period = C / gcd_i(C, V);
  s.active = kGnT / period * period;
  s.chunks = std::max<long>(1, (s.pieces + s.active - 1) / s.active);
  // two workgroups a CU over all images, as many as run at once (four: a stereo frame
  // at half resolution 10.2 + 13.7 us instead of 7.4 + 8.9); at least one chunk each
  s.blocks = (int)std::max<long>(1, std::min<long>(s.chunks, std::max(1, 512 / N)));
  return s;
}

__device__ __forceinline__ double wave_sum(double v, int width) {
  for (int o = width / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// Lanes that share one of `n` sums: the largest power of two <= min(64, kGnT / n).
__device__ __forceinline__ int lanes_per(int n) {
  int l = 1;
  while (l < 64 && 2 * l * n <= kGnT) l *= 2;
  return l;
}

// pass 1 of the forward: part[n][s][g] = (sum, sum of squares) of the block's
// values, 64-bit.
template <typename T>
__global__ void __launch_bounds__(kGnT) gn_stats_kernel(const T* __restrict__ x, int HW, int C, int G, Split sp,
                                                        double2* __restrict__ part) {
  constexpr int V = Elem<T>::V;
  __shared__ double2 red[kGnT * V];
  const int n = blockIdx.y, s = blockIdx.x, S = gridDim.x, t = threadIdx.x;
  const T* xb = x + (long)n * HW * C;
  const long c0 = sp.chunks * s / S, c1 = sp.chunks * (s + 1) / S;
  double s1[V], s2[V];
#pragma unroll
  for (int k = 0; k < V; ++k) s1[k] = s2[k] = 0.0;
  if (t < sp.active) {
    const long f1 = min(c1 * sp.active, sp.pieces);
    for (long f = c0 * sp.active + t; f < f1;) {
      float a[V], b[V], k0[V];
      const Piece<T> p0 = load_piece(xb + f * V);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        k0[k] = (float)p0.v[k];
        a[k] = b[k] = 0.f;
      }
      f += sp.active;
      int cnt = 1;
      while (cnt < kFlush && f < f1) {
        Piece<T> p[4];   // loads in flight
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (f + u * sp.active < f1) p[u] = load_piece(xb + (f + u * sp.active) * V);
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (f + u * sp.active < f1) {
            ++cnt;
#pragma unroll
            for (int k = 0; k < V; ++k) {
              const float d = (float)p[u].v[k] - k0[k];
              a[k] += d;
              b[k] = fmaf(d, d, b[k]);
            }
          }
        f += 4 * sp.active;
      }
#pragma unroll
      for (int k = 0; k < V; ++k) {   // about k0: sum = n k0 + a, squares = b + 2 k0 a + n k0^2
        const double q = k0[k], da = a[k];
        s1[k] += cnt * q + da;
        s2[k] += (double)b[k] + q * (2.0 * da + cnt * q);
      }
    }
    if (sp.tail && c1 == sp.chunks && sp.pieces % sp.active == t) {
      const Piece<T> p = load_tail(xb + sp.pieces * V, sp.tail);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const double q = (float)p.v[k];
        s1[k] += q;
        s2[k] += q * q;
      }
    }
  }
  // runs of r = gcd(cpg, V) values lie in one group: add them in registers
  const int cpg = C / G;
  int r = V;
  while (cpg % r) r /= 2;
  const int runs = V / r, span = C / r;            // run e of the active threads is run e % span of the channels
  const int copies = sp.active * V / C;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    double (&v)[V] = q ? s2 : s1;
    if (r >= 2) {
#pragma unroll
      for (int k = 0; k < V / 2; ++k) v[k] = v[2 * k] + v[2 * k + 1];
    }
    if (r >= 4) {
#pragma unroll
      for (int k = 0; k < V / 4; ++k) v[k] = v[2 * k] + v[2 * k + 1];
    }
    if (r >= 8) v[0] = v[0] + v[1];
  }
#pragma unroll
  for (int k = 0; k < V; ++k)
    if (k < runs && t < sp.active) red[t * runs + k] = make_double2(s1[k], s2[k]);
  __syncthreads();
  // a run of the channels over lanes of its own, then the runs and lanes of a group
  const int lanes = kGnT / span, run = t % span, ln = t / span;
  double u = 0.0, v = 0.0;
  if (ln < lanes)
#pragma unroll 4
    for (int i = ln; i < copies; i += lanes) {
      const double2 p = red[run + i * span];
      u += p.x;
      v += p.y;
    }
  __syncthreads();
  if (ln < lanes) red[run * lanes + ln] = make_double2(u, v);
  __syncthreads();
  const int L = lanes_per(G), g = t / L, l = t % L, terms = cpg / r * lanes;
  u = v = 0.0;
  if (g < G)
    for (int i = l; i < terms; i += L) {
      const double2 p = red[g * terms + i];
      u += p.x;
      v += p.y;
    }
  u = wave_sum(u, L);
  v = wave_sum(v, L);
  if (g < G && l == 0) part[((long)n * S + s) * G + g] = make_double2(u, v);
}

// mean and rstd of image n's groups from the S partials, in LDS (and to stats)
__device__ __forceinline__ void gn_finish_stats(const double2* part, int n, int S, int G, long M, float eps,
                                                double2* st, double2* stats_out) {
  const int t = threadIdx.x, L = lanes_per(G), g = t / L, l = t % L;
  double a = 0.0, b = 0.0;
  if (g < G)
#pragma unroll 4
    for (int s = l; s < S; s += L) {
      const double2 v = part[((long)n * S + s) * G + g];
      a += v.x;
      b += v.y;
    }
  a = wave_sum(a, L);
  b = wave_sum(b, L);
  if (g < G && l == 0) {
    const double mean = a / (double)M;
    double var = b / (double)M - mean * mean;
    if (var < 0.0) var = 0.0;   // (a NaN stays one)
    const double2 v = make_double2(mean, 1.0 / sqrt(var + (double)eps));
    st[g] = v;
    if (stats_out) stats_out[(long)n * G + g] = v;
  }
  __syncthreads();
}

__device__ __forceinline__ float relu(float v) { return v < 0.f ? 0.f : v; }   // passes a NaN on, as torch's

// SiLU's exponential and reciprocal are the hardware's: exp(-n) is off by |n| 2^-24
// (its argument's product with log2 e) and two units of fp32, the reciprocal by one,
// relative to silu(n) - which is exp(-|n|) |n| where |n| is large and negative.
template <int MODE>
__device__ __forceinline__ float gn_act(float n, float r) {
  if constexpr (MODE == kRelu) return relu(n);
  if constexpr (MODE == kResRelu) return relu(r + relu(n));
  if constexpr (MODE == kAddRelu) return relu(n + r);
  if constexpr (MODE == kSilu) return n * __builtin_amdgcn_rcpf(1.f + __expf(-n));
  return n;
}

// Channel constants: thread c < C makes channel c's (its integer divisions once, its
// parameters read early), the threads take their V from LDS (each thread for its own
// channels: one frame's second pass 8.2 us instead of 5.8).
struct ChanIn {
  float w, b;
  int g;
};
__device__ __forceinline__ ChanIn gn_channel(const void* w, const void* b, int wdt, int C, int cpg) {
  const int c = threadIdx.x;
  return c < C ? ChanIn{param(w, wdt, c, 1.f), param(b, wdt, c, 0.f), c / cpg} : ChanIn{0.f, 0.f, 0};
}
template <int V>
__device__ __forceinline__ void gn_take(float (&v)[V], const float* lds, int c0, int C) {
#pragma unroll
  for (int k = 0, c = c0; k < V; ++k) {
    v[k] = lds[c];
    c = c + 1 == C ? 0 : c + 1;
  }
}

// pass 2 of the forward
template <typename T, int MODE>
__global__ void __launch_bounds__(kGnT) gn_apply_kernel(const T* x, const T* res, T* out, const void* __restrict__ w,
                                                        const void* __restrict__ b, int wdt,
                                                        const double2* __restrict__ part, int S, int HW, int C, int G,
                                                        Split sp, float eps, double2* stats_out) {
  constexpr int V = Elem<T>::V;
  constexpr bool RES = MODE == kResRelu || MODE == kAddRelu;
  __shared__ double2 st[kGnMaxC];
  __shared__ float lds[3][kGnMaxC];
  constexpr int U = 4;
  const int n = blockIdx.y, t = threadIdx.x;
  const long base = (long)n * HW * C;
  const long c0 = sp.chunks * blockIdx.x / gridDim.x, c1 = sp.chunks * (blockIdx.x + 1) / gridDim.x;
  const long f1 = t < sp.active ? min(c1 * sp.active, sp.pieces) : 0;
  Piece<T> p[U], rp[U];
  auto load = [&](long f) {   // U pieces in flight a thread
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (f + u * sp.active < f1) {
        p[u] = load_piece(x + base + (f + u * sp.active) * V);
        if constexpr (RES) rp[u] = load_piece(res + base + (f + u * sp.active) * V);
      }
  };
  long f = c0 * sp.active + t;
  load(f);   // on their way while the statistics are added up
  const ChanIn ch = gn_channel(w, b, wdt, C, C / G);
  gn_finish_stats(part, n, S, G, (long)HW * (C / G), eps, st, blockIdx.x == 0 ? stats_out : nullptr);
  if (t < C) {   // y = (x - m) rw + b
    const double2 v = st[ch.g];
    lds[0][t] = (float)v.x;
    lds[1][t] = (float)(v.y * (double)ch.w);
    lds[2][t] = ch.b;
  }
  __syncthreads();
  if (t >= sp.active) return;
  float m[V], rw[V], bc[V];
  const int ct = (t * V) % C;
  gn_take(m, lds[0], ct, C);
  gn_take(rw, lds[1], ct, C);
  gn_take(bc, lds[2], ct, C);
  auto piece = [&](const Piece<T>& p, const Piece<T>& rp) {
    Piece<T> o;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float nn = fmaf((float)p.v[k] - m[k], rw[k], bc[k]);
      o.v[k] = (T)gn_act<MODE>(nn, RES ? (float)rp.v[k] : 0.f);
    }
    return o;
  };
  while (f < f1) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (f + u * sp.active < f1) store_piece(out + base + (f + u * sp.active) * V, piece(p[u], rp[u]));
    f += U * sp.active;
    load(f);
  }
  if (sp.tail && c1 == sp.chunks && sp.pieces % sp.active == t) {
    const long o = base + sp.pieces * V;
    const Piece<T> p = load_tail(x + o, sp.tail);
    Piece<T> rp;
    if constexpr (RES) rp = load_tail(res + o, sp.tail);
    store_tail(out + o, piece(p, rp), sp.tail);
  }
}

// The forward in one launch for small maps: one workgroup an image's group, whose
// pieces (cpg a multiple of V) stay in registers between the sums and the output.
// Bound by one trip to memory and the join of the sums.  Maps of 128 x 40 x 64 in
// fp16, 16 groups, us for 1, 4, 8, 12 of them: 7.1, 9.9, 13.4, 17.3; as two launches
// 10.3, 13.3, 14.2, 14.3.
constexpr int kSmallT = 1024, kSmallU = 4;
constexpr long kSmallBytes = 4 << 20;
template <typename T, int MODE>
__global__ void __launch_bounds__(kSmallT) gn_small_kernel(const T* x, const T* res, T* out,
                                                           const void* __restrict__ w, const void* __restrict__ b,
                                                           int wdt, int HW, int C, int G, float eps,
                                                           double2* __restrict__ stats_out) {
  constexpr int V = Elem<T>::V, U = kSmallU;
  constexpr bool RES = MODE == kResRelu || MODE == kAddRelu;
  __shared__ double2 red[kSmallT / 64];
  __shared__ __attribute__((aligned(16))) float rw[kGnMaxC], bc[kGnMaxC];
  const int n = blockIdx.y, g = blockIdx.x, t = threadIdx.x, cpg = C / G, per = cpg / V, total = HW * per;
  const long base = (long)n * HW * C + (long)g * cpg;
  Piece<T> p[U], rp[U];
  int at[U], part[U];   // a piece's place in the image, its first channel in the group
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int q = t + u * kSmallT;
    if (q < total) {
      const int pixel = q / per;
      part[u] = (q - pixel * per) * V;
      at[u] = pixel * C + part[u];
      p[u] = load_piece(x + base + at[u]);
      if constexpr (RES) rp[u] = load_piece(res + base + at[u]);
    }
  }
  const float wc = t < cpg ? param(w, wdt, g * cpg + t, 1.f) : 0.f;
  if (t < cpg) bc[t] = param(b, wdt, g * cpg + t, 0.f);
  double s1 = 0.0, s2 = 0.0;
  if (t < total) {   // about the thread's first value, as gn_stats_kernel
    const float k0 = (float)p[0].v[0];
    float a = 0.f, q2 = 0.f;
    int cnt = 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (t + u * kSmallT < total) {
        cnt += V;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float d = (float)p[u].v[k] - k0;
          a += d;
          q2 = fmaf(d, d, q2);
        }
      }
    const double q = k0, da = a;
    s1 = cnt * q + da;
    s2 = (double)q2 + q * (2.0 * da + cnt * q);
  }
  s1 = wave_sum(s1, 64);
  s2 = wave_sum(s2, 64);
  if ((t & 63) == 0) red[t / 64] = make_double2(s1, s2);
  __syncthreads();
  s1 = s2 = 0.0;
#pragma unroll
  for (int i = 0; i < kSmallT / 64; ++i) {
    s1 += red[i].x;
    s2 += red[i].y;
  }
  const double M = (double)HW * cpg, mean = s1 / M;
  double var = s2 / M - mean * mean;
  if (var < 0.0) var = 0.0;   // (a NaN stays one)
  const double rstd = 1.0 / sqrt(var + (double)eps);
  if (t == 0 && stats_out) stats_out[(long)n * G + g] = make_double2(mean, rstd);
  if (t < cpg) rw[t] = (float)(rstd * (double)wc);
  __syncthreads();
  const float m = (float)mean;
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (t + u * kSmallT < total) {
      Piece<T> o;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float nn = fmaf((float)p[u].v[k] - m, rw[part[u] + k], bc[part[u] + k]);
        o.v[k] = (T)gn_act<MODE>(nn, RES ? (float)rp[u].v[k] : 0.f);
      }
      store_piece(out + base + at[u], o);
    }
}

// dn and dres of one value (r: res, g: dy, n: the normed value).  tol = kTol times
// the largest 2 |b| + |m rw| of the thread's channels bounds n's fp32 error;
// returns whether a ReLU's argument is within that of zero (never where it is
// exact: channels with weight and bias 0, an image of zeros).
template <int MODE>
__device__ __forceinline__ bool gn_slope(float r, float g, float n, float tol, float& dn, float& dres) {
  dres = dn = g;
  if constexpr (MODE == kSilu) {
    const float sg = __builtin_amdgcn_rcpf(1.f + __expf(-n));
    dn = g * sg * (1.f + n * (1.f - sg));
  } else if constexpr (MODE == kRelu) {
    dn = n > 0.f ? g : 0.f;
    return fabsf(n) < tol;
  } else if constexpr (MODE == kResRelu) {
    const float pre = r + fmaxf(n, 0.f);
    dres = pre > 0.f ? g : 0.f;
    dn = n > 0.f ? dres : 0.f;
    return fabsf(n) < tol || (n > 0.f && fabsf(pre) < fmaf(kTol, fabsf(r), tol));   // (n < 0: pre is r itself)
  } else if constexpr (MODE == kAddRelu) {
    const float pre = n + r;
    dn = dres = pre > 0.f ? g : 0.f;
    return fabsf(pre) < fmaf(kTol, fabsf(r), tol);
  }
  return false;
}

// dn and dres of a piece of cnt values at x + o.  The 64-bit decisions, a branch
// hardly ever taken, are made one value at a time with everything read again and
// kept as two bit masks: unrolled, they took more registers than all the rest.
template <typename T, int MODE>
__device__ __forceinline__ void gn_slopes(const float (&nn)[Elem<T>::V], const Piece<T>& rp, const Piece<T>& gp,
                                          float tol, const T* x, const T* res, long o, int cnt, const double2* st,
                                          const void* w, const void* b, int wdt, int C, int cpg,
                                          float (&dn)[Elem<T>::V], float (&dr)[Elem<T>::V]) {
  constexpr int V = Elem<T>::V;
  constexpr bool RES = MODE == kResRelu || MODE == kAddRelu;
  bool near = false;
#pragma unroll
  for (int k = 0; k < V; ++k)
    near |= gn_slope<MODE>(RES ? (float)rp.v[k] : 0.f, (float)gp.v[k], nn[k], tol, dn[k], dr[k]);
  if constexpr (MODE != kNone && MODE != kSilu) {
    if (__builtin_expect(near, 0)) {
      int t = threadIdx.x;
      asm volatile("" : "+v"(t));   // (or its channel arithmetic moves out of the loop)
      int c = (t * V) % C;
      unsigned on_n = 0, on_o = 0;
#pragma unroll 1
      for (int k = 0; k < cnt; ++k) {
        const double2 sg = st[c / cpg];
        const double n = ((double)(float)x[o + k] - sg.x) * (sg.y * (double)param(w, wdt, c, 1.f)) +
                         (double)param(b, wdt, c, 0.f);
        const double rv = RES ? (double)(float)res[o + k] : 0.0;
        on_n |= (unsigned)(n > 0.0) << k;
        on_o |= (unsigned)((MODE == kResRelu ? rv + fmax(n, 0.0) : n + rv) > 0.0) << k;
        c = c + 1 == C ? 0 : c + 1;
      }
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float g = (float)gp.v[k];
        if constexpr (RES) dr[k] = on_o >> k & 1 ? g : 0.f;
        if constexpr (MODE == kAddRelu) dn[k] = dr[k];
        if constexpr (MODE != kAddRelu) dn[k] = on_n >> k & 1 ? dr[k] : 0.f;
      }
    }
  }
}

// pass 1 of the backward: per block the channel sums of dn and dn xhat
// (cpart[n][s][c]) and the group sums of w dn and w dn xhat (gpart[n][s][g]);
// writes dres.
template <typename T, int MODE>
__global__ void __launch_bounds__(kGnT, 4) gn_bwd_stats_kernel(const T* __restrict__ x, const T* __restrict__ res,
                                                            const T* __restrict__ dy, T* __restrict__ dres,
                                                            const void* __restrict__ w, const void* __restrict__ b,
                                                            int wdt, const double2* __restrict__ stats, int HW, int C,
                                                            int G, Split sp, double2* __restrict__ cpart,
                                                            double2* __restrict__ gpart) {
  constexpr int V = Elem<T>::V;
  constexpr bool RES = MODE == kResRelu || MODE == kAddRelu;
  __shared__ double red[2][V][kGnT + 8];   // value k of thread t at [k][t]; + 8: the channels read across the k below
  __shared__ double2 sum[kGnT];
  const int n = blockIdx.y, s = blockIdx.x, S = gridDim.x, t = threadIdx.x;
  const int cpg = C / G;
  const double2* st = stats + (long)n * G;
  // channel constants: xhat = (x - m) rs, n = xhat wc + bc
  float m[V], rs[V], wc[V], bc[V], a1[V], a2[V], tol = 0.f;
  {
    float (&lds)[4][kGnMaxC] = *reinterpret_cast<float (*)[4][kGnMaxC]>(&red[0][0][0]);   // free again before the sums
    const ChanIn ch = gn_channel(w, b, wdt, C, cpg);
    if (t < C) {
      const double2 v = st[ch.g];
      lds[0][t] = (float)v.x;
      lds[1][t] = (float)v.y;
      lds[2][t] = ch.w;
      lds[3][t] = ch.b;
    }
    __syncthreads();
    const int ct = (t * V) % C;
    gn_take(m, lds[0], ct, C);
    gn_take(rs, lds[1], ct, C);
    gn_take(wc, lds[2], ct, C);
    gn_take(bc, lds[3], ct, C);
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < V; ++k) {
    tol = fmaxf(tol, kTol * (2.f * fabsf(bc[k]) + fabsf(m[k] * rs[k] * wc[k])));
    a1[k] = a2[k] = 0.f;
    red[0][k][t] = red[1][k][t] = 0.0;
  }
  // from fp32 to 64 bits, in LDS: in registers the kernel would spill
  auto flush = [&]() {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      red[0][k][t] += (double)a1[k];
      red[1][k][t] += (double)a2[k];
      a1[k] = a2[k] = 0.f;
    }
  };
  const long base = (long)n * HW * C;
  const long c0 = sp.chunks * s / S, c1 = sp.chunks * (s + 1) / S;
  const long f1 = min(c1 * sp.active, sp.pieces);
  auto piece = [&](const Piece<T>& p, const Piece<T>& rp, const Piece<T>& gp, long at, int cnt) {
    float xh[V], nn[V], dn[V], dr[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      xh[k] = ((float)p.v[k] - m[k]) * rs[k];
      nn[k] = fmaf(xh[k], wc[k], bc[k]);
    }
    gn_slopes<T, MODE>(nn, rp, gp, tol, x, res, at, cnt, st, w, b, wdt, C, cpg, dn, dr);
    Piece<T> o;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      if (k < cnt) {
        a1[k] += dn[k];
        a2[k] = fmaf(dn[k], xh[k], a2[k]);
      }
      o.v[k] = (T)dr[k];
    }
    return o;
  };
  if (t < sp.active) {
    // two pieces' loads in flight a thread
    int cnt = 0;
    for (long f = c0 * sp.active + t; f < f1; f += 2 * sp.active) {
      if (cnt == kFlush) flush(), cnt = 0;
      cnt += 2;
      Piece<T> p[2], gp[2], rp[2];
      const bool two = f + sp.active < f1;
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (u == 0 || two) {
          const long o = base + (f + u * sp.active) * V;
          p[u] = load_piece(x + o), gp[u] = load_piece(dy + o);
          if constexpr (RES) rp[u] = load_piece(res + o);
        }
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (u == 0 || two) {
          const long at = base + (f + u * sp.active) * V;
          const Piece<T> o = piece(p[u], rp[u], gp[u], at, V);
          if constexpr (RES) store_piece(dres + at, o);
        }
    }
    if (sp.tail && c1 == sp.chunks && sp.pieces % sp.active == t) {
      const long o0 = base + sp.pieces * V;
      const Piece<T> p = load_tail(x + o0, sp.tail), gp = load_tail(dy + o0, sp.tail);
      Piece<T> rp;
      if constexpr (RES) rp = load_tail(res + o0, sp.tail);
      const Piece<T> o = piece(p, rp, gp, o0, sp.tail);
      if constexpr (RES) store_tail(dres + o0, o, sp.tail);
    }
    flush();
  }
  __syncthreads();
  // channel c: the flat values c, c + C, ... of the active threads, over lanes of
  // its own (l slow: neighbouring threads read neighbouring channels)
  const int copies = sp.active * V / C;
  const int L = max(1, kGnT / C), l = t / C, c = t % C;
  double u = 0.0, v = 0.0;
  if (l < L)
    for (int i = l; i < copies; i += L) {
      const int f = c + i * C;
      u += red[0][f % V][f / V];
      v += red[1][f % V][f / V];
    }
  sum[t] = make_double2(u, v);
  __syncthreads();
  if (t < C) {
    for (int i = 1; i < L; ++i) {
      u += sum[t + i * C].x;
      v += sum[t + i * C].y;
    }
    cpart[((long)n * S + s) * C + t] = make_double2(u, v);
    const double wc = (double)param(w, wdt, t, 1.f);
    sum[t] = make_double2(u * wc, v * wc);
  }
  __syncthreads();
  if (t < G) {
    u = v = 0.0;
    for (int i = 0; i < cpg; ++i) {
      u += sum[t * cpg + i].x;
      v += sum[t * cpg + i].y;
    }
    gpart[((long)n * S + s) * G + t] = make_double2(u, v);
  }
}

// pass 2 of the backward: dx; the grid's last row of workgroups (blockIdx.y ==
// N) adds up the channel sums to dw and db instead.
template <typename T, int MODE>
__global__ void __launch_bounds__(kGnT, 4) gn_bwd_apply_kernel(const T* __restrict__ x, const T* __restrict__ dyr,
                                                            T* __restrict__ dx, const void* __restrict__ w,
                                                            const void* __restrict__ b, int wdt,
                                                            const double2* __restrict__ stats, int N, int HW, int C,
                                                            int G, Split sp, int S, const double2* __restrict__ cpart,
                                                            const double2* __restrict__ gpart, void* __restrict__ dw,
                                                            void* __restrict__ db) {
  constexpr int V = Elem<T>::V;
  __shared__ double2 sm[kGnT];
  const int t = threadIdx.x;
  if (blockIdx.y == N) {
    // 16 channels a workgroup, 32 lanes over the N S partials of each
    const int l = t / 16;
    for (int c0 = blockIdx.x * 16; c0 < C; c0 += gridDim.x * 16) {
      const int c = c0 + t % 16;
      double u = 0.0, v = 0.0;
      if (c < C)
#pragma unroll 4
        for (int i = l; i < N * S; i += kGnT / 16) {
          const double2 p = cpart[(long)i * C + c];
          u += p.x;
          v += p.y;
        }
      __syncthreads();
      sm[t] = make_double2(u, v);
      __syncthreads();
      if (t < 16 && c < C) {
        u = v = 0.0;
        for (int i = 0; i < kGnT / 16; ++i) {
          u += sm[t + 16 * i].x;
          v += sm[t + 16 * i].y;
        }
        if (wdt == 1) {
          if (dw) static_cast<float*>(dw)[c] = (float)v;
          if (db) static_cast<float*>(db)[c] = (float)u;
        } else if (wdt == 0) {
          if (dw) static_cast<_Float16*>(dw)[c] = (_Float16)(float)v;
          if (db) static_cast<_Float16*>(db)[c] = (_Float16)(float)u;
        } else {
          if (dw) static_cast<__bf16*>(dw)[c] = (__bf16)(float)v;
          if (db) static_cast<__bf16*>(db)[c] = (__bf16)(float)u;
        }
      }
    }
    return;
  }
  // the images in the other order: the last ones are still in the cache
  const int cpg = C / G, n = N - 1 - blockIdx.y;
  const double2* st = stats + (long)n * G;
  const long base = (long)n * HW * C;
  const long c0 = sp.chunks * blockIdx.x / gridDim.x, c1 = sp.chunks * (blockIdx.x + 1) / gridDim.x;
  const long f1 = t < sp.active ? min(c1 * sp.active, sp.pieces) : 0;
  Piece<T> p[2], gp[2];
  auto load = [&](long f) {   // two pieces in flight a thread
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (f + u * sp.active < f1) {
        const long o = base + (f + u * sp.active) * V;
        p[u] = load_piece(x + o), gp[u] = load_piece(dyr + o);
      }
  };
  long f = c0 * sp.active + t;
  load(f);   // on their way while the sums are added up
  __shared__ float lds[5][kGnMaxC];
  const ChanIn ch = gn_channel(w, b, wdt, C, cpg);
  {
    const int L = lanes_per(G), g = t / L, l = t % L;
    double u = 0.0, v = 0.0;
    if (g < G)
#pragma unroll 4
      for (int s = l; s < S; s += L) {
        const double2 p = gpart[((long)n * S + s) * G + g];
        u += p.x;
        v += p.y;
      }
    u = wave_sum(u, L);
    v = wave_sum(v, L);
    const double M = (double)HW * cpg;
    if (g < G && l == 0) sm[g] = make_double2(u / M, v / M);
    __syncthreads();
    if (t < C) {
      const double2 ms = st[ch.g], kk = sm[ch.g];
      lds[0][t] = (float)ms.x;
      lds[1][t] = (float)(ms.y * (double)ch.w);
      lds[2][t] = ch.b;
      lds[3][t] = (float)(ms.y * kk.x);
      lds[4][t] = (float)(ms.y * ms.y * kk.y);
    }
    __syncthreads();
  }
  if (t >= sp.active) return;
  // dx = rstd w dn - rstd (k1 + xhat k2): per channel rw = rstd w, q1 = rstd k1, q2 = rstd^2 k2
  float m[V], rw[V], bc[V], q1[V], q2[V], tol = 0.f;
  const int ct = (t * V) % C;
  gn_take(m, lds[0], ct, C);
  gn_take(rw, lds[1], ct, C);
  gn_take(bc, lds[2], ct, C);
  gn_take(q1, lds[3], ct, C);
  gn_take(q2, lds[4], ct, C);
#pragma unroll
  for (int k = 0; k < V; ++k) tol = fmaxf(tol, kTol * (2.f * fabsf(bc[k]) + fabsf(m[k] * rw[k])));
  // the outer ReLU's slope is in dyr (= dres) already: what is left is mode 0's
  // ReLU (mode 1's inner one), or SiLU's slope
  constexpr int LEFT = MODE == kResRelu ? (int)kRelu : MODE == kAddRelu ? (int)kNone : MODE;
  auto piece = [&](const Piece<T>& p, const Piece<T>& gp, long at, int cnt) {
    float d[V], nn[V], dn[V], dr[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      d[k] = (float)p.v[k] - m[k];
      nn[k] = fmaf(d[k], rw[k], bc[k]);
    }
    gn_slopes<T, LEFT>(nn, gp, gp, tol, x, nullptr, at, cnt, st, w, b, wdt, C, cpg, dn, dr);
    Piece<T> o;
#pragma unroll
    for (int k = 0; k < V; ++k) o.v[k] = (T)(fmaf(dn[k], rw[k], -fmaf(d[k], q2[k], q1[k])));
    return o;
  };
  while (f < f1) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (f + u * sp.active < f1) {
        const long at = base + (f + u * sp.active) * V;
        store_piece(dx + at, piece(p[u], gp[u], at, V));
      }
    f += 2 * sp.active;
    load(f);
  }
  if (sp.tail && c1 == sp.chunks && sp.pieces % sp.active == t) {
    const long o0 = base + sp.pieces * V;
    const Piece<T> p = load_tail(x + o0, sp.tail), gp = load_tail(dyr + o0, sp.tail);
    store_tail(dx + o0, piece(p, gp, o0, sp.tail), sp.tail);
  }
}

inline int gn_vec(int dtype) { return dtype == 1 ? 4 : 8; }

// Whether the forward is one launch: the group's values fit the registers of a
// workgroup, and the maps are small (the 16-B pieces of neighbouring groups share
// lines that each workgroup fetches again).
inline bool gn_is_small(int dtype, int N, int HW, int C, int G) {
  const int V = gn_vec(dtype), cpg = C / G;
  return cpg % V == 0 && (long)HW * (cpg / V) <= kSmallT * kSmallU &&
         (long)N * HW * C * (16 / V) <= kSmallBytes;
}

int gn_check(const char* what, int dtype, int wdtype, int N, int HW, int C, int G, int mode) {
  if (dtype != 0 && dtype != 1 && dtype != 3)
    return fail(kInvalidArgument, std::string(what) + ": dtype must be float16, float32 or bfloat16");
  if (wdtype != 1 && wdtype != dtype)
    return fail(kInvalidArgument, std::string(what) + ": weight and bias must be float32 or of x's type");
  if (N < 0 || HW < 0 || C <= 0 || C > kGnMaxC || G <= 0 || C % G || mode < 0 || mode > 4)
    return fail(kInvalidArgument, std::string(what) + ": bad arguments (0 < C <= 512, C % groups == 0, mode 0..4)");
  if (N > 65534) return fail(kUnsupported, std::string(what) + ": more than 65534 images");
  return kOk;
}

}  // namespace

}  // namespace droid

using namespace droid;

#define GN_MODES(T, KERNEL, ...)                         \
  switch (mode) {                                        \
    case kRelu: KERNEL(T, kRelu, __VA_ARGS__); break;       \
    case kResRelu: KERNEL(T, kResRelu, __VA_ARGS__); break; \
    case kAddRelu: KERNEL(T, kAddRelu, __VA_ARGS__); break; \
    case kNone: KERNEL(T, kNone, __VA_ARGS__); break;       \
    default: KERNEL(T, kSilu, __VA_ARGS__); break;          \
  }
#define GN_TYPES(KERNEL, ...)                                  \
  if (dtype == 0) {                                            \
    GN_MODES(_Float16, KERNEL, __VA_ARGS__)                    \
  } else if (dtype == 1) {                                     \
    GN_MODES(float, KERNEL, __VA_ARGS__)                       \
  } else {                                                     \
    GN_MODES(__bf16, KERNEL, __VA_ARGS__)                      \
  }

extern "C" {

size_t droid_group_norm_workspace(int dtype, int N, int HW, int C, int G, int backward) {
  if (gn_check("group_norm_workspace", dtype, 1, N, HW, C, G, 0) != kOk || N == 0 || HW == 0) return 0;
  if (!backward && gn_is_small(dtype, N, HW, C, G)) return 0;
  const Split sp = gn_split(N, HW, C, gn_vec(dtype));
  return (size_t)N * sp.blocks * (G + (backward ? C : 0)) * sizeof(double2);
}

int droid_group_norm_act(int dtype, const void* x, const void* res, void* out, const void* weight, const void* bias,
                         int wdtype, void* stats, int N, int HW, int C, int G, int mode, float eps, void* ws,
                         size_t ws_bytes, hipStream_t stream) {
  if (const int st = gn_check("group_norm_act", dtype, wdtype, N, HW, C, G, mode)) return st;
  if (N == 0 || HW == 0) return kOk;
  const bool need_res = mode == kResRelu || mode == kAddRelu;
  if (!x || !out || (need_res && !res)) return fail(kInvalidArgument, "group_norm_act: null map");
  if (gn_is_small(dtype, N, HW, C, G)) {
#define GN_SMALL(T, M, ...)                                                                                          \
  gn_small_kernel<T, M><<<dim3(G, N), kSmallT, 0, stream>>>((const T*)x, (const T*)res, (T*)out, weight, bias, wdtype, \
                                                            HW, C, G, eps, (double2*)stats)
    GN_TYPES(GN_SMALL, 0)
#undef GN_SMALL
    DROID_LAUNCH_CHECK();
    return kOk;
  }
  if (!ws || ws_bytes < droid_group_norm_workspace(dtype, N, HW, C, G, 0))
    return fail(kInvalidArgument, "group_norm_act: workspace too small");
  const Split sp = gn_split(N, HW, C, gn_vec(dtype));
  double2* part = static_cast<double2*>(ws);
  const dim3 grid(sp.blocks, N);
#define GN_STATS(T) gn_stats_kernel<T><<<grid, kGnT, 0, stream>>>((const T*)x, HW, C, G, sp, part)
  if (dtype == 0) GN_STATS(_Float16);
  else if (dtype == 1) GN_STATS(float);
  else GN_STATS(__bf16);
#undef GN_STATS
  DROID_LAUNCH_CHECK();
#define GN_APPLY(T, M, ...)                                                                                          \
  gn_apply_kernel<T, M><<<grid, kGnT, 0, stream>>>((const T*)x, (const T*)res, (T*)out, weight, bias, wdtype, part, \
                                                   sp.blocks, HW, C, G, sp, eps, (double2*)stats)
  GN_TYPES(GN_APPLY, 0)
#undef GN_APPLY
  DROID_LAUNCH_CHECK();
  return kOk;
}

int droid_group_norm_act_backward(int dtype, const void* x, const void* res, const void* dy, const void* weight,
                                  const void* bias, int wdtype, const void* stats, void* dx, void* dres, void* dweight,
                                  void* dbias, int N, int HW, int C, int G, int mode, void* ws, size_t ws_bytes,
                                  hipStream_t stream) {
  if (const int st = gn_check("group_norm_act_backward", dtype, wdtype, N, HW, C, G, mode)) return st;
  if (N == 0 || HW == 0) return kOk;
  const bool need_res = mode == kResRelu || mode == kAddRelu;
  if (!x || !dy || !dx || !stats || (need_res && (!res || !dres)))
    return fail(kInvalidArgument, "group_norm_act_backward: null map");
  if (!ws || ws_bytes < droid_group_norm_workspace(dtype, N, HW, C, G, 1))
    return fail(kInvalidArgument, "group_norm_act_backward: workspace too small");
  const Split sp = gn_split(N, HW, C, gn_vec(dtype));
  double2* gpart = static_cast<double2*>(ws);
  double2* cpart = gpart + (size_t)N * sp.blocks * G;
  const double2* st = static_cast<const double2*>(stats);
#define GN_BSTATS(T, M, ...)                                                                                        \
  gn_bwd_stats_kernel<T, M><<<dim3(sp.blocks, N), kGnT, 0, stream>>>((const T*)x, (const T*)res, (const T*)dy,      \
                                                                     (T*)dres, weight, bias, wdtype, st, HW, C, G,  \
                                                                     sp, cpart, gpart)
  GN_TYPES(GN_BSTATS, 0)
#undef GN_BSTATS
  DROID_LAUNCH_CHECK();
#define GN_BAPPLY(T, M, ...)                                                                                          \
  gn_bwd_apply_kernel<T, M><<<dim3(sp.blocks, N + (dweight || dbias ? 1 : 0)), kGnT, 0, stream>>>(                    \
      (const T*)x, (const T*)(need_res ? dres : dy), (T*)dx, weight, bias, wdtype, st, N, HW, C, G, sp, sp.blocks, \
      cpart, gpart, dweight, dbias)
  GN_TYPES(GN_BAPPLY, 0)
#undef GN_BAPPLY
  DROID_LAUNCH_CHECK();
  return kOk;
}

}  // extern "C"
