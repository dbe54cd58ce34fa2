// Rotary positions with several axes (line, image, video) on the q and k rows of an attention.
//
// The first 2 * P of a head's D dims are P pairs (x1, x2); pair p belongs to one axis and is turned by
// angle = position[token][axis(p)] * theta^(-j / n) (j-th of the axis' n pairs):
//   y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin
// The backward is the turn by the negative angle.  Dims from 2 * P on pass unchanged.
//
// Bound by memory: 2 * elements * size bytes, every element read and written once: 65536 tokens, 16 + 4 heads of 128, bf16
// take 148 us a direction, 4.5 TB/s (a large copy: 4.9).  A workgroup forms the
// sines and cosines of its tokens once in LDS and uses them for all heads of q and k.  Angles are kept in
// turns and reduced to (-1/2, 1/2] in fp64 (a position of 10^5 leaves an fp32 angle with 2 decimal digits).
#include "ogv_common.h"

#include <math.h>

namespace ogv {

constexpr int ROT_PAIRS = 64;   // head_dim <= 128

struct RotTensor {
  const void* x;
  void* y;
  long row_in, head_in, row_out, head_out;
  int heads;
};

struct RotArgs {
  RotTensor t[2];
  const void* pos;
  int M, axes, D, P, interleaved, pos_float;
  float sign;
  double turns[ROT_PAIRS];           // theta^(-j / n) / (2 pi)
  unsigned char axis[ROT_PAIRS];
};

// V elements of each half of the pairs (or of interleaved pairs) per item; a workgroup's items are counted in 32 bits
template <typename T, int V, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(const RotArgs a, int TB) {
  extern __shared__ float2 cs[];   // [TB][P]: cos, sin
  const long m0 = (long)blockIdx.x * TB;
  const int nt = (int)min((long)TB, a.M - m0), P = a.P;
  for (int i = threadIdx.x; i < nt * P; i += 256) {
    const int tok = i / P, p = i - tok * P;
    const long at = (m0 + tok) * a.axes + a.axis[p];
    const double pos = a.pos_float ? (double)((const float*)a.pos)[at] : (double)((const int*)a.pos)[at];
    double turn = pos * a.turns[p];
    turn -= rint(turn);
    float s, c;
    sincospif(2.f * (float)turn, &s, &c);
    cs[i] = make_float2(c, a.sign * s);
  }
  __syncthreads();
  // items of a token and head: pair chunks, then the chunks that pass
  const int np = INTER ? 2 * P / V : P / V, per = np + (a.D - 2 * P) / V;
  const int h0 = a.t[0].heads, heads = h0 + a.t[1].heads;
  for (int i = threadIdx.x; i < nt * heads * per; i += 256) {
    const int th = i / per, ch = i - th * per, tok = th / heads, hh = th - tok * heads;
    const RotTensor& t = a.t[hh >= h0];
    const int h = hh >= h0 ? hh - h0 : hh;
    const T* x = (const T*)t.x + (m0 + tok) * t.row_in + h * t.head_in;
    T* y = (T*)t.y + (m0 + tok) * t.row_out + h * t.head_out;
    const float2* w = cs + tok * P;
    if (ch >= np) {
      const int d = 2 * P + (ch - np) * V;
      float u[V];
      load_vec<T, V>(x + d, u);
      store_vec<T, V>(y + d, u);
    } else if constexpr (INTER) {
      float u[V], o[V];
      load_vec<T, V>(x + ch * V, u);
#pragma unroll
      for (int e = 0; e < V / 2; ++e) {
        const float2 z = w[ch * (V / 2) + e];
        o[2 * e] = u[2 * e] * z.x - u[2 * e + 1] * z.y;
        o[2 * e + 1] = u[2 * e + 1] * z.x + u[2 * e] * z.y;
      }
      store_vec<T, V>(y + ch * V, o);
    } else {
      float u[V], v[V], o1[V], o2[V];
      load_vec<T, V>(x + ch * V, u);
      load_vec<T, V>(x + P + ch * V, v);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 z = w[ch * V + e];
        o1[e] = u[e] * z.x - v[e] * z.y;
        o2[e] = v[e] * z.x + u[e] * z.y;
      }
      store_vec<T, V>(y + ch * V, o1);
      store_vec<T, V>(y + P + ch * V, o2);
    }
  }
}

template <typename T>
static void rotary_launch(const RotArgs& a, bool vec, int TB, hipStream_t s) {
  const unsigned nb = cdiv(a.M, TB);
  const size_t lds = (size_t)TB * a.P * sizeof(float2);
  if (a.interleaved) {
    if (vec) rotary_kernel<T, 8, true><<<nb, 256, lds, s>>>(a, TB);
    else rotary_kernel<T, 2, true><<<nb, 256, lds, s>>>(a, TB);
  } else {
    if (vec) rotary_kernel<T, 8, false><<<nb, 256, lds, s>>>(a, TB);
    else rotary_kernel<T, 1, false><<<nb, 256, lds, s>>>(a, TB);
  }
}

}  // namespace ogv

using namespace ogv;

extern "C" int ogv_axial_rotary(const void* q, void* q_out, const void* k, void* k_out, const void* positions,
                                const ogv_rotary_desc* d, ogv_dtype dt, void* stream) {
  OGV_REQUIRE(d && q && q_out && positions, "ogv_axial_rotary: null pointer");
  OGV_REQUIRE(dt == OGV_F32 || dt == OGV_BF16, "ogv_axial_rotary: bad dtype %d", (int)dt);
  OGV_REQUIRE(d->M >= 0 && d->heads[0] > 0 && d->heads[1] >= 0, "ogv_axial_rotary: bad shape M=%d heads=%d, %d", d->M,
              d->heads[0], d->heads[1]);
  OGV_REQUIRE(d->heads[1] == 0 || (k && k_out), "ogv_axial_rotary: null k");
  OGV_REQUIRE(d->axes > 0 && d->axes <= OGV_ROTARY_AXES, "ogv_axial_rotary: axes=%d (1..%d)", d->axes, OGV_ROTARY_AXES);
  OGV_REQUIRE(d->theta > 0. && __builtin_isfinite(d->theta), "ogv_axial_rotary: theta must be positive and finite");
  RotArgs a = {};
  int P = 0;
  for (int x = 0; x < d->axes; ++x) {
    OGV_REQUIRE(d->pairs[x] > 0 && d->pairs[x] <= ROT_PAIRS - P, "ogv_axial_rotary: bad sections (pairs per axis)");
    for (int j = 0; j < d->pairs[x]; ++j, ++P) {
      a.turns[P] = pow(d->theta, -(double)j / d->pairs[x]) * 0.15915494309189533577;
      a.axis[P] = (unsigned char)x;
    }
  }
  OGV_REQUIRE(2 * P <= d->D && d->D <= 2 * ROT_PAIRS && d->D % 2 == 0,
              "ogv_axial_rotary: head_dim=%d must be even, <= %d and hold 2 * %d turned dims", d->D, 2 * ROT_PAIRS, P);
  if (d->M == 0) return OGV_OK;
  const size_t es = dt == OGV_BF16 ? 2 : 4;
  const void* in[2] = {q, k};
  void* out[2] = {q_out, k_out};
  bool vec = d->D % 8 == 0 && P % (d->interleaved ? 4 : 8) == 0;
  for (int i = 0; i < 2; ++i) {
    a.t[i] = RotTensor{in[i], out[i], (long)d->row_in[i], (long)d->head_in[i], (long)d->row_out[i], (long)d->head_out[i],
                       d->heads[i]};
    if (!d->heads[i]) continue;
    const int64_t s[4] = {d->row_in[i], d->head_in[i], d->row_out[i], d->head_out[i]};
    for (int64_t v : s) {
      OGV_REQUIRE(v >= 0, "ogv_axial_rotary: negative stride");
      vec = vec && v * es % 16 == 0;
      OGV_REQUIRE(!d->interleaved || v % 2 == 0, "ogv_axial_rotary: strides of interleaved pairs must be even");
    }
    OGV_REQUIRE((uintptr_t)in[i] % (d->interleaved ? 2 * es : es) == 0 && (uintptr_t)out[i] % (d->interleaved ? 2 * es : es) == 0,
                "ogv_axial_rotary: misaligned pointer");
    vec = vec && (uintptr_t)in[i] % 16 == 0 && (uintptr_t)out[i] % 16 == 0;
  }
  a.pos = positions, a.M = d->M, a.axes = d->axes, a.D = d->D, a.P = P, a.interleaved = d->interleaved;
  a.pos_float = d->pos_float, a.sign = d->inverse ? -1.f : 1.f;
  const int TB = 8, V = vec ? 8 : d->interleaved ? 2 : 1;
  const long items = (long)(d->M < TB ? d->M : TB) * ((long)d->heads[0] + d->heads[1]) * ((d->interleaved ? 2 * P : P) / V + (d->D - 2 * P) / V);
  OGV_REQUIRE(items < (1L << 31) - 256, "ogv_axial_rotary: too many heads (%d + %d)", d->heads[0], d->heads[1]);
  if (dt == OGV_BF16) rotary_launch<bf16>(a, vec, TB, as_stream(stream));
  else rotary_launch<float>(a, vec, TB, as_stream(stream));
  return check_launch("ogv_axial_rotary");
}
