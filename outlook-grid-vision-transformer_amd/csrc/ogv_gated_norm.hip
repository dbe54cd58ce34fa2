// The end of a residual half-block and the norm that begins the next one, in one pass over the rows:
//
//   n = N_post(f) (or f)        y = alpha * x + s_b * gate * n        h = N_pre(y) (none: only y)
//
// N(v) = (v - mean) * rstd * w + b (layer) or v * rstd * w + b with rstd = 1 / sqrt(mean(v^2) + eps) (rms);
// gate per channel or per sample and channel, s_b a factor per sample (DropPath).  h is formed from y before
// y is rounded, and the backward forms the same y again from f and x, so no gradient carries that rounding:
//   dY = dy + N_pre'(dh)   dx = alpha dY   dn = s_b gate dY   df = N_post'(dn)
//   dgate = sum s_b n dY   (dw, db) of a norm = sums of (g vhat, g) over the rows
//   N'(g) = rstd (g w - [mean(g w)] - vhat mean(g w vhat))        ([.]: layer only)
//
// Bound by memory: forward f, x -> y, h (4 rows of C), backward f, x, dy, dh -> df, dx (6): 65536 rows of 768, bf16, layer
// norms on both sides take 90 us and 133 us, 4.5 TB/s (a large copy: 4.9); 12800 rows of 331, fp32, 15 and 26 us; wider
// rows were not timed.  The backward loads the next row while it works on one.  A row belongs to G lanes (a part of a
// wave, a wave, or a workgroup) that hold it through every reduction, in registers as far as these go.  Of rows above 512
// channels read in vectors, the backward's registers leave two waves to a SIMD at 520 to 768 in bf16 with a gate per
// channel (which, with two sums for three gradients, took the case above from 355 to 133 us) and at 1032 to 2048, else one.
// Above 4096 channels it spills: 97 registers (bf16) or 224 (fp32), 221 or 343 with a gate per sample, 515 to 631 where
// single columns are read.
// Column sums: each lane adds its columns over the workgroup's rows, one partial row per workgroup, then they are added
// in a fixed order: no atomics.
#include "ogv_common.h"

#include <initializer_list>

namespace ogv {

enum { NK_NONE = OGV_NORM_NONE, NK_LAYER = OGV_NORM_LAYER, NK_RMS = OGV_NORM_RMS };

struct GnArgs {
  const void *f, *x, *dy, *dh;
  void *y, *h, *df, *dx;
  const float *gate, *rs, *w0, *b0, *w1, *b1;   // 0: post, 1: pre
  float* stats;     // [M][4]: post mean, post rstd, pre mean, pre rstd
  float *part, *gpart;   // backward column sums: [blocks][4][C]; per-sample gate: [units][C]
  long M;
  int C, k0, k1, rps;
  int S, nch;       // gate samples (1: the gate has no samples), row chunks per sample
  long rows_s, rows_c;   // rows per sample, rows per chunk
  float alpha, eps0, eps1;
};

// sum over the G lanes of a row; G > 64: the whole workgroup owns one row (every thread reaches this)
template <int G> __device__ __forceinline__ float row_sum(float v, float* red) {
  if constexpr (G <= 64) {
    return group_sum<G>(v);
  } else {
    static_assert(G == 256, "a row is a part of a wave, a wave or a workgroup");
    v = group_sum<64>(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return ((red[0] + red[1]) + red[2]) + red[3];
  }
}

// v -> (v - mean) * rstd in place (columns outside C hold 0 on entry and are not counted)
template <int G, int E>
__device__ __forceinline__ void normalise(float (&v)[E], const bool (&in)[E], int kind, float invC, float eps,
                                          float& mean, float& rstd, float* red) {
  float s = 0.f;
  mean = 0.f;
  if (kind == NK_LAYER) {
#pragma unroll
    for (int e = 0; e < E; ++e) s += v[e];
    mean = row_sum<G>(s, red) * invC;
  }
  s = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    v[e] = in[e] ? v[e] - mean : 0.f;
    s = fmaf(v[e], v[e], s);
  }
  rstd = rsqrtf(row_sum<G>(s, red) * invC + eps);
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] *= rstd;
}

// NV vectors of VEC columns per lane, lane q of the row's G holding columns (v * G + q) * VEC + i
template <typename T, int G, int NV, int VEC>
__global__ __launch_bounds__(256) void gated_norm_fwd_kernel(const GnArgs a) {
  constexpr int E = NV * VEC, R = 256 / G;
  __shared__ float red[4];
  const int lg = threadIdx.x % G, C = a.C;
  const float invC = 1.f / (float)C;
  bool in[E];
  float gw[E], w0[E], b0[E], w1[E], b1[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = ((e / VEC) * G + lg) * VEC + e % VEC, cc = c < C ? c : 0;
    in[e] = c < C;
    gw[e] = a.gate && a.S == 1 ? a.gate[cc] : 1.f;
    w0[e] = a.w0 ? a.w0[cc] : 1.f;
    b0[e] = a.b0 ? a.b0[cc] : 0.f;
    w1[e] = a.w1 ? a.w1[cc] : 1.f;
    b1[e] = a.b1 ? a.b1[cc] : 0.f;
  }
  for (long row = (long)blockIdx.x * R + threadIdx.x / G; row < a.M; row += (long)gridDim.x * R) {
    float f[E], x[E], sc[E], mean, rstd;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + lg) * VEC, cc = c < C ? c : 0;
      load_vec<T, VEC>((const T*)a.f + row * C + cc, f + v * VEC);
      load_vec<T, VEC>((const T*)a.x + row * C + cc, x + v * VEC);
    }
    const float rs = a.rs ? a.rs[row / a.rps] : 1.f;
#pragma unroll
    for (int e = 0; e < E; ++e) sc[e] = rs * gw[e];
    if (a.S > 1) {
      const float* g = a.gate + (row / a.rows_s) * C;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = ((e / VEC) * G + lg) * VEC + e % VEC;
        sc[e] = rs * g[c < C ? c : 0];
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = in[e] ? f[e] : 0.f;
    if (a.k0 != NK_NONE) {
      normalise<G, E>(f, in, a.k0, invC, a.eps0, mean, rstd, red);
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = fmaf(f[e], w0[e], b0[e]);
      if (a.stats && lg == 0) a.stats[row * 4] = mean, a.stats[row * 4 + 1] = rstd;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = in[e] ? fmaf(sc[e], f[e], a.alpha * x[e]) : 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (in[v * VEC]) store_vec<T, VEC>((T*)a.y + row * C + (v * G + lg) * VEC, x + v * VEC);
    if (a.k1 != NK_NONE) {
      normalise<G, E>(x, in, a.k1, invC, a.eps1, mean, rstd, red);
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = fmaf(x[e], w1[e], b1[e]);
#pragma unroll
      for (int v = 0; v < NV; ++v)
        if (in[v * VEC]) store_vec<T, VEC>((T*)a.h + row * C + (v * G + lg) * VEC, x + v * VEC);
      if (a.stats && lg == 0) a.stats[row * 4 + 2] = mean, a.stats[row * 4 + 3] = rstd;
    }
  }
}

// dv of N: rstd * (gw - [mean(gw)] - vhat * mean(gw * vhat)); columns outside C hold 0
template <int G, int E>
__device__ __forceinline__ void norm_back(float (&gw)[E], const float (&vh)[E], int kind, float invC, float rstd, float* red) {
  float s1 = 0.f, s2 = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) s1 += gw[e], s2 = fmaf(gw[e], vh[e], s2);
  const float m1 = kind == NK_LAYER ? row_sum<G>(s1, red) * invC : 0.f;
  const float m2 = row_sum<G>(s2, red) * invC;
#pragma unroll
  for (int e = 0; e < E; ++e) gw[e] = rstd * (gw[e] - m1 - vh[e] * m2);
}

// column sums of the workgroup: over the 256 / G row slots of each column, into out[C]
template <int G, int NV, int VEC>
__device__ __forceinline__ void flush_sums(float (&s)[NV * VEC], float* __restrict__ out, int C, float* buf) {
  constexpr int E = NV * VEC;
  const int lg = threadIdx.x % G, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if constexpr (G < 256) {
    if constexpr (G < 64) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        for (int o = G; o < 64; o <<= 1) s[e] += __shfl_xor(s[e], o, 64);
    }
    constexpr int L = G < 64 ? G : 64;   // buf: [4][E * L]
    __syncthreads();
    if (lane < L) {
#pragma unroll
      for (int e = 0; e < E; ++e) buf[(wave * E + e) * L + lane] = s[e];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < E * L; i += 256) {
      const int e = i / L, q = i - e * L;
      const int c = ((e / VEC) * G + q) * VEC + e % VEC;
      if (c < C) out[c] = ((buf[i] + buf[E * L + i]) + buf[2 * E * L + i]) + buf[3 * E * L + i];
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = ((e / VEC) * G + lg) * VEC + e % VEC;
      if (c < C) out[c] = s[e];
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) s[e] = 0.f;
}

// The raw values of a row that the backward reads, loaded one row ahead of their use.
template <typename T, int G, int NV, int VEC> struct BackRow {
  RawVec<T, VEC> f[NV], x[NV], dy[NV], dh[NV];
  float4 st;
  float rs;
  __device__ __forceinline__ void load(const GnArgs& a, long row, int lg) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + lg) * VEC;
      const long at = row * a.C + (c < a.C ? c : 0);
      f[v].load((const T*)a.f + at);
      x[v].load((const T*)a.x + at);
      if (a.dy) dy[v].load((const T*)a.dy + at);
      if (a.dh) dh[v].load((const T*)a.dh + at);
    }
    st = *reinterpret_cast<const float4*>(a.stats + row * 4);
    rs = a.rs ? a.rs[row / a.rps] : 1.f;
  }
};

// Column sums kept per lane: A = sum s_b dY fhat and B = sum s_b dY (fhat = f without a post norm) give every gradient
// of the branch's side -- dgate = w A + b B, dw = gate A, db = gate B -- so a gate per channel needs no third sum, and a
// gate per sample (SMP) closes A and B into s0, t0 at a sample's end.  s1, t1: the pre norm's.
template <typename T, int G, int NV, int VEC, bool SMP>
__global__ __launch_bounds__(256) void gated_norm_bwd_kernel(const GnArgs a) {
  constexpr int E = NV * VEC, R = 256 / G, L = G < 64 ? G : 64;
  __shared__ float red[4];
  __shared__ float buf[G < 256 ? 4 * E * L : 1];
  const int lg = threadIdx.x % G, C = a.C;
  const float invC = 1.f / (float)C;
  bool in[NV];
  float gw[E], w0[E], b0[E], w1[E];
  float A[E], B[E], s1[E], t1[E], s0[SMP ? E : 1], t0[SMP ? E : 1];
#pragma unroll
  for (int v = 0; v < NV; ++v) in[v] = (v * G + lg) * VEC < C;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = ((e / VEC) * G + lg) * VEC + e % VEC, cc = c < C ? c : 0;
    gw[e] = a.gate && !SMP ? a.gate[cc] : 1.f;
    w0[e] = a.w0 ? a.w0[cc] : 1.f;
    b0[e] = a.b0 ? a.b0[cc] : 0.f;
    w1[e] = a.w1 ? a.w1[cc] : 1.f;
    A[e] = B[e] = s1[e] = t1[e] = 0.f;
    if constexpr (SMP) s0[e] = t0[e] = 0.f;
  }
  const long units = (long)a.S * a.nch;
  for (long u = blockIdx.x; u < units; u += gridDim.x) {
    const long smp = u / a.nch, ch = u - smp * a.nch;
    const long beg = smp * a.rows_s + ch * a.rows_c, end = min(beg + a.rows_c, (smp + 1) * a.rows_s);
    if constexpr (SMP) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = ((e / VEC) * G + lg) * VEC + e % VEC;
        gw[e] = a.gate[smp * C + (c < C ? c : 0)];
      }
    }
    long row = beg + threadIdx.x / G;
    BackRow<T, G, NV, VEC> next;
    if (row < end) next.load(a, row, lg);
    for (; row < end; row += R) {
      float f[E], x[E], dY[E];
      const float4 st = next.st;
      const float rs = next.rs;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        next.f[v].unpack(f + v * VEC);
        next.x[v].unpack(x + v * VEC);
      }
      float dh[E], dy[E];
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        if (a.dy) next.dy[v].unpack(dy + v * VEC);
        if (a.dh) next.dh[v].unpack(dh + v * VEC);
      }
      next.load(a, min(row + R, end - 1), lg);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        f[e] = in[e / VEC] ? (a.k0 != NK_NONE ? (f[e] - st.x) * st.y : f[e]) : 0.f;   // fhat
        dY[e] = 0.f;
      }
      if (a.dh) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          x[e] = in[e / VEC] ? (fmaf(rs * gw[e], fmaf(f[e], w0[e], b0[e]), a.alpha * x[e]) - st.z) * st.w : 0.f;   // yhat
          const float g = in[e / VEC] ? dh[e] : 0.f;
          s1[e] = fmaf(g, x[e], s1[e]);
          t1[e] += g;
          dY[e] = g * w1[e];
        }
        norm_back<G, E>(dY, x, a.k1, invC, st.w, red);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (a.dy) dY[e] += in[e / VEC] ? dy[e] : 0.f;
        x[e] = a.alpha * dY[e];
        dY[e] *= rs;
        A[e] = fmaf(dY[e], f[e], A[e]);
        B[e] += dY[e];
        dY[e] *= gw[e];   // dn
      }
#pragma unroll
      for (int v = 0; v < NV; ++v)
        if (in[v]) store_vec<T, VEC>((T*)a.dx + row * C + (v * G + lg) * VEC, x + v * VEC);
      if (a.k0 != NK_NONE) {
#pragma unroll
        for (int e = 0; e < E; ++e) dY[e] *= in[e / VEC] ? w0[e] : 0.f;
        norm_back<G, E>(dY, f, a.k0, invC, st.y, red);
      }
#pragma unroll
      for (int v = 0; v < NV; ++v)
        if (in[v]) store_vec<T, VEC>((T*)a.df + row * C + (v * G + lg) * VEC, dY + v * VEC);
    }
    if constexpr (SMP) {
      float d[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        d[e] = fmaf(w0[e], A[e], b0[e] * B[e]);
        s0[e] = fmaf(gw[e], A[e], s0[e]);
        t0[e] = fmaf(gw[e], B[e], t0[e]);
        A[e] = B[e] = 0.f;
      }
      flush_sums<G, NV, VEC>(d, a.gpart + u * C, C, buf);
    }
  }
  float* out = a.part + (long)blockIdx.x * 4 * C;
  if constexpr (SMP) {
    flush_sums<G, NV, VEC>(s0, out, C, buf);
    flush_sums<G, NV, VEC>(t0, out + C, C, buf);
  } else {
    flush_sums<G, NV, VEC>(A, out, C, buf);
    flush_sums<G, NV, VEC>(B, out + C, C, buf);
  }
  flush_sums<G, NV, VEC>(s1, out + 2 * C, C, buf);
  flush_sums<G, NV, VEC>(t1, out + 3 * C, C, buf);
}

// The partial rows part [rows][4][C] added in a fixed order into sums [5][C] = dgate, d pre_w, d pre_b, d post_w, d post_b,
// and dgate [S][C] from the samples' row chunks.  Workgroup: 64 columns of one pair of sums, 16 waves on every 16th row.
__global__ __launch_bounds__(1024) void gated_norm_sum_kernel(const GnArgs a, float* __restrict__ sums, float* __restrict__ dgate,
                                                              int rows, int colblocks) {
  const int C = a.C, bx = blockIdx.x;
  if (bx >= 2 * colblocks) {
    const long i = (long)(bx - 2 * colblocks) * 1024 + threadIdx.x;
    if (i >= (long)a.S * C) return;
    const long s = i / C, c = i - s * C;
    float v = 0.f;
    for (int j = 0; j < a.nch; ++j) v += a.gpart[(s * a.nch + j) * C + c];
    dgate[i] = v;
    return;
  }
  __shared__ float red[2][16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, pair = bx / colblocks;
  const int c = (bx - pair * colblocks) * 64 + lane, cc = min(c, C - 1);
  const float* p = a.part + 2L * pair * C + cc;
  float x = 0.f, y = 0.f;
#pragma unroll 8
  for (int r = wave; r < rows; r += 16) {
    x += p[(long)r * 4 * C];
    y += p[(long)r * 4 * C + C];
  }
  red[0][wave][lane] = x, red[1][wave][lane] = y;
  __syncthreads();
  if (wave || c >= C) return;
  x = y = 0.f;
#pragma unroll
  for (int w = 0; w < 16; ++w) x += red[0][w][lane], y += red[1][w][lane];
  if (pair) {
    sums[C + c] = x, sums[2 * C + c] = y;
  } else if (a.S > 1) {
    sums[3 * C + c] = x, sums[4 * C + c] = y;
  } else {
    const float g = a.gate ? a.gate[c] : 1.f, w = a.w0 ? a.w0[c] : 1.f, b = a.b0 ? a.b0[c] : 0.f;
    sums[c] = fmaf(w, x, b * y), sums[3 * C + c] = g * x, sums[4 * C + c] = g * y;
  }
}

// Lanes per row and columns per lane: vectors where the channel count and the pointers allow them; up to 1024
// channels a row stays inside a wave (its reductions need no barrier), above that a workgroup owns it.
struct GnPlan {
  int G, NV, VEC;
};

static bool gn_plan(int C, bool vec, GnPlan& p) {
  p.VEC = vec && C % 8 == 0 ? (C > 512 && C <= 768 ? 4 : 8) : 1;
  const int n = C / p.VEC;   // vectors per row
  if (p.VEC == 4) {          // 64 lanes x 3 vectors of 4
    p.G = 64, p.NV = 3;
    return true;
  }
  if (p.VEC == 8) {
    p.G = 2;
    while (p.G < n && p.G < 64) p.G <<= 1;
    if (C > 1024) p.G = 256;
    p.NV = (n + p.G - 1) / p.G;
    if (p.NV == 3) p.NV = 4;
    return p.NV <= 4;
  }
  p.G = n <= 512 ? 64 : 256;
  p.NV = (n + p.G - 1) / p.G;
  for (int nv : {1, 2, 4, 6, 8, 16, 32})
    if (p.NV <= nv) {
      p.NV = nv;
      return true;
    }
  return false;
}

constexpr long GN_BLOCKS = 512;   // workgroups of the backward (two to a CU), and partial rows of its column sums

static void gn_units(long M, long samples, const GnPlan& p, GnArgs& a, long& blocks) {
  a.S = (int)samples;
  a.rows_s = M / samples;
  const long R = 256 / p.G;
  long nch = (GN_BLOCKS + samples - 1) / samples;
  const long most = (a.rows_s + R - 1) / R;
  if (nch > most) nch = most;
  a.rows_c = (a.rows_s + nch - 1) / nch;
  a.nch = (int)((a.rows_s + a.rows_c - 1) / a.rows_c);
  const long units = samples * a.nch;
  blocks = units < GN_BLOCKS ? units : GN_BLOCKS;
}

template <typename T, int G, int NV, int VEC>
static void gn_run(const GnArgs& a, bool bwd, long blocks, hipStream_t s) {
  if (bwd && a.S > 1) gated_norm_bwd_kernel<T, G, NV, VEC, true><<<(unsigned)blocks, 256, 0, s>>>(a);
  else if (bwd) gated_norm_bwd_kernel<T, G, NV, VEC, false><<<(unsigned)blocks, 256, 0, s>>>(a);
  else gated_norm_fwd_kernel<T, G, NV, VEC><<<(unsigned)blocks, 256, 0, s>>>(a);
}

template <typename T> static void gn_dispatch(const GnPlan& p, const GnArgs& a, bool bwd, long blocks, hipStream_t s) {
  if (p.VEC == 4) return gn_run<T, 64, 3, 4>(a, bwd, blocks, s);
  if (p.VEC == 8) {
    switch (p.G) {
      case 2: return gn_run<T, 2, 1, 8>(a, bwd, blocks, s);
      case 4: return gn_run<T, 4, 1, 8>(a, bwd, blocks, s);
      case 8: return gn_run<T, 8, 1, 8>(a, bwd, blocks, s);
      case 16: return gn_run<T, 16, 1, 8>(a, bwd, blocks, s);
      case 32: return gn_run<T, 32, 1, 8>(a, bwd, blocks, s);
      case 64:
        if (p.NV == 1) return gn_run<T, 64, 1, 8>(a, bwd, blocks, s);
        return gn_run<T, 64, 2, 8>(a, bwd, blocks, s);
      default:
        if (p.NV == 1) return gn_run<T, 256, 1, 8>(a, bwd, blocks, s);
        if (p.NV == 2) return gn_run<T, 256, 2, 8>(a, bwd, blocks, s);
        return gn_run<T, 256, 4, 8>(a, bwd, blocks, s);
    }
  }
  if (p.G == 64) {
    if (p.NV == 1) return gn_run<T, 64, 1, 1>(a, bwd, blocks, s);
    if (p.NV == 2) return gn_run<T, 64, 2, 1>(a, bwd, blocks, s);
    if (p.NV == 4) return gn_run<T, 64, 4, 1>(a, bwd, blocks, s);
    if (p.NV == 6) return gn_run<T, 64, 6, 1>(a, bwd, blocks, s);
    return gn_run<T, 64, 8, 1>(a, bwd, blocks, s);
  }
  if (p.NV <= 4) return gn_run<T, 256, 4, 1>(a, bwd, blocks, s);
  if (p.NV <= 8) return gn_run<T, 256, 8, 1>(a, bwd, blocks, s);
  if (p.NV == 16) return gn_run<T, 256, 16, 1>(a, bwd, blocks, s);
  return gn_run<T, 256, 32, 1>(a, bwd, blocks, s);
}

static int gn_check(const char* what, const ogv_gated_norm_desc* d, ogv_dtype dt) {
  OGV_REQUIRE(d, "%s: null descriptor", what);
  OGV_REQUIRE(dt == OGV_F32 || dt == OGV_BF16, "%s: bad dtype %d", what, (int)dt);
  OGV_REQUIRE(d->M > 0 && d->C > 0 && d->C <= 8192, "%s: bad shape M=%d C=%d (need 1 <= C <= 8192)", what, d->M, d->C);
  OGV_REQUIRE(d->post >= 0 && d->post <= 2 && d->pre >= 0 && d->pre <= 2, "%s: bad norm kind %d, %d", what, d->post, d->pre);
  OGV_REQUIRE(d->samples >= 1 && d->M % d->samples == 0, "%s: M=%d rows do not divide into %d samples", what, d->M, d->samples);
  OGV_REQUIRE(d->rps >= 1, "%s: rps must be >= 1", what);
  return OGV_OK;
}

static bool gn_vec(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if ((uintptr_t)p & 15) return false;
  return true;
}

static void gn_fill(const ogv_gated_norm_desc* d, const float* gate, const float* rs, const float* const* w, GnArgs& a) {
  a = GnArgs{};
  a.M = d->M, a.C = d->C, a.k0 = d->post, a.k1 = d->pre, a.rps = d->rps;
  a.alpha = d->alpha, a.eps0 = d->post_eps, a.eps1 = d->pre_eps;
  a.gate = gate, a.rs = rs, a.w0 = w[0], a.b0 = w[1], a.w1 = w[2], a.b1 = w[3];
}

}  // namespace ogv

using namespace ogv;

extern "C" int ogv_gated_norm_fwd(const void* f, const void* x, const float* gate, const float* rs, const float* post_w,
                                  const float* post_b, const float* pre_w, const float* pre_b, void* y, void* h,
                                  float* stats, const ogv_gated_norm_desc* d, ogv_dtype dt, void* stream) {
  if (int rc = gn_check("ogv_gated_norm_fwd", d, dt)) return rc;
  OGV_REQUIRE(f && x && y && (d->pre == NK_NONE || h), "ogv_gated_norm_fwd: null pointer");
  const float* w[4] = {post_w, post_b, pre_w, pre_b};
  GnArgs a;
  gn_fill(d, gate, rs, w, a);
  a.f = f, a.x = x, a.y = y, a.h = h, a.stats = stats;
  a.S = gate ? d->samples : 1, a.rows_s = d->M / a.S;
  GnPlan p;
  OGV_REQUIRE(gn_plan(d->C, gn_vec({f, x, y, h}), p), "ogv_gated_norm_fwd: C=%d unsupported", d->C);
  const long R = 256 / p.G, nb = (d->M + R - 1) / R, blocks = nb < 2048 ? nb : 2048;
  if (dt == OGV_BF16) gn_dispatch<bf16>(p, a, false, blocks, as_stream(stream));
  else gn_dispatch<float>(p, a, false, blocks, as_stream(stream));
  return check_launch("ogv_gated_norm_fwd");
}

extern "C" size_t ogv_gated_norm_bwd_ws_bytes(const ogv_gated_norm_desc* d, ogv_dtype dt) {
  if (gn_check("ogv_gated_norm_bwd_ws_bytes", d, dt) != OGV_OK) return 0;
  size_t most = 0;
  for (bool vec : {false, true}) {   // the pointers are not known here: the larger plan
    GnPlan p;
    GnArgs a;
    long blocks;
    if (!gn_plan(d->C, vec, p)) continue;
    for (long samples : {1L, (long)d->samples}) {   // (nor whether there is a gate)
      gn_units(d->M, samples, p, a, blocks);
      const size_t n = (size_t)blocks * 4 * d->C + (a.S > 1 ? (size_t)a.S * a.nch * d->C : 0);
      if (n > most) most = n;
    }
  }
  return most * sizeof(float);
}

extern "C" int ogv_gated_norm_bwd(const void* dy, const void* dh, const void* f, const void* x, const float* gate,
                                  const float* rs, const float* post_w, const float* post_b, const float* pre_w,
                                  const float* pre_b, const float* stats, void* df, void* dx, float* sums, float* dgate,
                                  void* ws, const ogv_gated_norm_desc* d, ogv_dtype dt, void* stream) {
  if (int rc = gn_check("ogv_gated_norm_bwd", d, dt)) return rc;
  OGV_REQUIRE(f && x && stats && df && dx && sums && ws && (dy || dh), "ogv_gated_norm_bwd: null pointer");
  OGV_REQUIRE(!dh || d->pre != NK_NONE, "ogv_gated_norm_bwd: dh without a pre norm");
  OGV_REQUIRE(d->samples == 1 || !gate || dgate, "ogv_gated_norm_bwd: a gate per sample needs dgate");
  const float* w[4] = {post_w, post_b, pre_w, pre_b};
  GnArgs a;
  gn_fill(d, gate, rs, w, a);
  a.f = f, a.x = x, a.dy = dy, a.dh = dh, a.df = df, a.dx = dx, a.stats = const_cast<float*>(stats);
  GnPlan p;
  OGV_REQUIRE(gn_plan(d->C, gn_vec({f, x, dy, dh, df, dx}), p), "ogv_gated_norm_bwd: C=%d unsupported", d->C);
  long blocks;
  gn_units(d->M, gate ? d->samples : 1, p, a, blocks);
  a.part = (float*)ws;
  a.gpart = a.part + (size_t)blocks * 4 * d->C;
  hipStream_t s = as_stream(stream);
  if (dt == OGV_BF16) gn_dispatch<bf16>(p, a, true, blocks, s);
  else gn_dispatch<float>(p, a, true, blocks, s);
  const int cb = (int)cdiv(d->C, 64);
  gated_norm_sum_kernel<<<2 * cb + (a.S > 1 ? cdiv((long)a.S * d->C, 1024) : 0), 1024, 0, s>>>(a, sums, dgate, (int)blocks, cb);
  return check_launch("ogv_gated_norm_bwd");
}
