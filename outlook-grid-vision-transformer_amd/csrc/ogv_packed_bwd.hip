// Attention over packed sequences, backward, from the forward's lse (probabilities are recomputed):
//
//   p_rj = exp(s_rj - lse_r)     delta_r = sum_d do_rd o_rd      dp_rj = do_r . v_j
//   ds_rj = p_rj (dp_rj - delta_r)
//   dq_r = scale sum_j ds_rj k_j      dk_j = scale sum_r ds_rj q_r      dv_j = sum_r p_rj do_r
//
// Two kernels, each owning the rows it writes, so no sum depends on the order of workgroups: dq walks the
// keys of a row block (and forms delta), dk / dv walk the rows -- of all query heads that share the key head --
// of a key block.  That computes the scores and dp twice (7 products for 5) and needs no atomics and no zeroed
// accumulators.  P and dS are rounded to bf16 for their products; scores, dp, delta and sums are fp32.
#include "ogv_packed.h"

#include <initializer_list>

namespace ogv {

int packed_check(const char* what, const ogv_packed_desc* d, ogv_dtype dt);
void packed_args(const ogv_packed_desc* d, PackedArgs& a);
bool aligned16(std::initializer_list<const void*> ps);

constexpr float BLOG2E = 1.4426950408889634f;

template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64) void packed_dq_kernel(const PackedArgs a) {
  using F = Frag<T, D>;
  constexpr int BM = 32 * NW, BN = 32, NT = NW * 64;
  constexpr int RB = F::RB, NC = F::NC, KK = F::KK, E = F::E;
  __shared__ __attribute__((aligned(16))) char Ks[BN * RB];
  __shared__ __attribute__((aligned(16))) char Vs[BN * RB];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hf = lane >> 5, c = lane & 31;

  int h, t;
  if (!head_tile(a.d, a.hkv, a.tiles, h, t)) return;
  const Seq sq = find_tile(a.cu_q, a.B, a.Mq, a.G, BM, a.tiles - 1 - t, lane);
  const int k0 = cu_at(a.cu_k, sq.b, a.Mk), lk = max(cu_at(a.cu_k, sq.b + 1, a.Mk) - k0, 0);
  const int rows = sq.len * a.G, r0 = sq.tile * BM;
  const int store_rows = sq.b == a.B - 1 ? (a.Mq - sq.start) * a.G : rows;
  if (r0 >= store_rows) return;
  const int off = lk - sq.len;
  int kend = r0 < rows ? lk : 0;
  if (a.causal && kend) kend = max(0, min(lk, group_div(min(r0 + BM, rows) - 1, a.G, a.gmagic) + off + 1));

  const int r = r0 + wave * 32 + c, pos = group_div(r, a.G, a.gmagic), hg = r - pos * a.G;
  const bool live = r < rows;
  const int lim = live ? (a.causal ? min(lk - 1, pos + off) : lk - 1) : -1;
  const long orow = (long)(sq.start + (live ? pos : 0)) * a.hq + h * a.G + hg;
  Chunk qf[KK], gf[KK];
  float delta = 0.f;
  {
    const long row = sq.start + (live ? pos : 0), head = h * a.G + hg;
    const T* qp = (const T*)a.q + row * a.rq + head * a.hsq;
    const T* gp = (const T*)a.dout + row * a.rdo + head * a.hsdo;
    const T* op = (const T*)a.o + row * a.ro + head * a.hso;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const int d = (2 * kk + hf) * E;
      qf[kk] = gf[kk] = zero_chunk();
      if (live && d < a.D) {
        qf[kk].u = *reinterpret_cast<const uint4*>(qp + d);
        gf[kk].u = *reinterpret_cast<const uint4*>(gp + d);
        Chunk oc;
        oc.u = *reinterpret_cast<const uint4*>(op + d);
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int e = 0; e < 8; ++e) delta = fmaf((float)gf[kk].h[e], (float)oc.h[e], delta);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) delta = fmaf(gf[kk].f[e], oc.f[e], delta);
        }
      }
    }
  }
  delta += __shfl_xor(delta, 32, 64);
  if (live && hf == 0) a.delta[orow] = delta;
  // a row that sees nothing has lse = -inf: its weights are masked below, +inf keeps the others' at 0
  float lse2 = live ? a.lse[orow] * BLOG2E : INFINITY;
  if (lse2 == -INFINITY) lse2 = INFINITY;
  f32x16 dq[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db) dq[db] = f32x16{};
  const float c2 = a.scale * BLOG2E;
  const T* kb = (const T*)a.k + (long)k0 * a.rk + (long)h * a.hsk;
  const T* vb = (const T*)a.v + (long)k0 * a.rv + (long)h * a.hsv;

  for (int key0 = 0; key0 < kend; key0 += BN) {
    __syncthreads();
#pragma unroll
    for (int n = 0; n < (BN * NC + NT - 1) / NT; ++n) {
      const int idx = tid + n * NT;
      if (BN * NC % NT == 0 || idx < BN * NC) {
        const int row = idx / NC, ch = idx - row * NC;
        Chunk kc = zero_chunk(), vc = zero_chunk();
        if (key0 + row < lk && ch * E < a.D) {
          kc.u = *reinterpret_cast<const uint4*>(kb + (long)(key0 + row) * a.rk + ch * E);
          vc.u = *reinterpret_cast<const uint4*>(vb + (long)(key0 + row) * a.rv + ch * E);
        }
        const int at = row * RB + ((ch ^ swz<RB>(row)) << 4);
        *reinterpret_cast<uint4*>(Ks + at) = kc.u;
        *reinterpret_cast<uint4*>(Vs + at) = vc.u;
      }
    }
    __syncthreads();
    f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      mfma_step<T>(lds_chunk<RB>(Ks, c, 2 * kk + hf), qf[kk], s);
      mfma_step<T>(lds_chunk<RB>(Vs, c, 2 * kk + hf), gf[kk], dp);
    }
    const bool masked = !__all(key0 + BN - 1 <= lim);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float p = __builtin_amdgcn_exp2f(fmaf(s[i], c2, -lse2)) * (dp[i] - delta);
      if (masked && key0 + 8 * (i / 4) + 4 * hf + i % 4 > lim) p = 0.f;
      s[i] = p;
    }
    accum_xt<T, D>(Ks, 0, s, dq, lane);
  }

  if (r >= store_rows) return;
  T* qp = (T*)a.dq + (long)(sq.start + pos) * a.rdq + (long)(h * a.G + hg) * a.hsdq;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = db * 32 + 8 * g + 4 * hf;
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = dq[db][4 * g + e] * a.scale;
      if (d < a.D) store_vec<T, 4>(qp + d, x);
    }
}

template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64) void packed_dkv_kernel(const PackedArgs a) {
  using F = Frag<T, D>;
  constexpr int BM = 32 * NW, BN = 32, NT = NW * 64;   // BM keys of the workgroup, BN rows per step
  constexpr int RB = F::RB, NC = F::NC, KK = F::KK, E = F::E;
  __shared__ __attribute__((aligned(16))) char Qs[BN * RB];
  __shared__ __attribute__((aligned(16))) char Gs[BN * RB];
  __shared__ __attribute__((aligned(16))) float Ls[BN], Ds[BN];
  __shared__ __attribute__((aligned(16))) int Lim[BN];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hf = lane >> 5, c = lane & 31;

  int h, t;
  if (!head_tile(a.d, a.hkv, a.tiles, h, t)) return;
  const Seq sk = find_tile(a.cu_k, a.B, a.Mk, 1, BM, t, lane);
  const int q0 = cu_at(a.cu_q, sk.b, a.Mq), lq = max(cu_at(a.cu_q, sk.b + 1, a.Mq) - q0, 0);
  const int j0 = sk.tile * BM, off = sk.len - lq, rows = lq * a.G;
  const int store_keys = sk.b == a.B - 1 ? a.Mk - sk.start : sk.len;
  if (j0 >= store_keys) return;
  int rbeg = 0, rend = j0 < sk.len ? rows : 0;
  if (a.causal) rbeg = (int)(min((long)rend, (long)max(0, j0 - off) * a.G) / BN) * BN;   // rows that see key j0 or later

  const int j = j0 + wave * 32 + c;
  const bool live = j < sk.len;
  Chunk kf[KK], vf[KK];
  {
    const T* kp = (const T*)a.k + (long)(sk.start + (live ? j : 0)) * a.rk + (long)h * a.hsk;
    const T* vp = (const T*)a.v + (long)(sk.start + (live ? j : 0)) * a.rv + (long)h * a.hsv;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const int d = (2 * kk + hf) * E;
      kf[kk] = vf[kk] = zero_chunk();
      if (live && d < a.D) {
        kf[kk].u = *reinterpret_cast<const uint4*>(kp + d);
        vf[kk].u = *reinterpret_cast<const uint4*>(vp + d);
      }
    }
  }
  f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db) dk[db] = f32x16{}, dv[db] = f32x16{};
  const float c2 = a.scale * BLOG2E;
  const T* qb = (const T*)a.q + (long)q0 * a.rq + (long)h * a.G * a.hsq;
  const T* gb = (const T*)a.dout + (long)q0 * a.rdo + (long)h * a.G * a.hsdo;

  for (int rt = rbeg; rt < rend; rt += BN) {
    __syncthreads();
#pragma unroll
    for (int n = 0; n < (BN * NC + NT - 1) / NT; ++n) {
      const int idx = tid + n * NT;
      if (BN * NC % NT == 0 || idx < BN * NC) {
        const int row = idx / NC, ch = idx - row * NC, r = rt + row;
        Chunk qc = zero_chunk(), gc = zero_chunk();
        if (r < rows && ch * E < a.D) {
          const int pos = group_div(r, a.G, a.gmagic), hg = r - pos * a.G;
          qc.u = *reinterpret_cast<const uint4*>(qb + (long)pos * a.rq + (long)hg * a.hsq + ch * E);
          gc.u = *reinterpret_cast<const uint4*>(gb + (long)pos * a.rdo + (long)hg * a.hsdo + ch * E);
        }
        const int at = row * RB + ((ch ^ swz<RB>(row)) << 4);
        *reinterpret_cast<uint4*>(Qs + at) = qc.u;
        *reinterpret_cast<uint4*>(Gs + at) = gc.u;
      }
    }
    for (int i = tid; i < BN; i += NT) {
      const int r = rt + i;
      float lse = INFINITY, delta = 0.f;   // a row that sees nothing, or none: weights exp2(-inf) = 0
      int lim = -1;
      if (r < rows) {
        const int pos = group_div(r, a.G, a.gmagic);
        const long orow = (long)(q0 + pos) * a.hq + h * a.G + (r - pos * a.G);
        lse = a.lse[orow] * BLOG2E;
        if (lse == -INFINITY) lse = INFINITY;
        delta = a.delta[orow];
        lim = a.causal ? pos + off : sk.len;
      }
      Ls[i] = lse, Ds[i] = delta, Lim[i] = lim;
    }
    __syncthreads();
    f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      mfma_step<T>(lds_chunk<RB>(Qs, c, 2 * kk + hf), kf[kk], s);
      mfma_step<T>(lds_chunk<RB>(Gs, c, 2 * kk + hf), vf[kk], dp);
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 lse = *reinterpret_cast<const f32x4*>(Ls + 8 * g + 4 * hf);
      const f32x4 del = *reinterpret_cast<const f32x4*>(Ds + 8 * g + 4 * hf);
      const int4 lim = *reinterpret_cast<const int4*>(Lim + 8 * g + 4 * hf);
      const int li[4] = {lim.x, lim.y, lim.z, lim.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 4 * g + e;
        float p = __builtin_amdgcn_exp2f(fmaf(s[i], c2, -lse[e]));
        if (j > li[e]) p = 0.f;
        s[i] = p;
        dp[i] = p * (dp[i] - del[e]);
      }
    }
    accum_xt<T, D>(Gs, 0, s, dv, lane);
    accum_xt<T, D>(Qs, 0, dp, dk, lane);
  }

  if (j >= store_keys) return;
  T* kp = (T*)a.dk + (long)(sk.start + j) * a.rdk + (long)h * a.hsdk;
  T* vp = (T*)a.dv + (long)(sk.start + j) * a.rdv + (long)h * a.hsdv;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = db * 32 + 8 * g + 4 * hf;
      float x[4], y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = dk[db][4 * g + e] * a.scale, y[e] = dv[db][4 * g + e];
      if (d < a.D) {
        store_vec<T, 4>(kp + d, x);
        store_vec<T, 4>(vp + d, y);
      }
    }
}

template <typename T, int D>
static void bwd_launch(PackedArgs a, hipStream_t s) {
  const long rows = (long)a.Mq * a.G;
  const int nwq = rows >= 96L * a.B ? 4 : 1, nwk = a.Mk >= 96L * a.B ? 4 : 1;
  a.tiles = (int)(rows / (32 * nwq)) + a.B;
  a.d = deal(a.hkv, a.tiles);
  const unsigned nq = deal_grid(a.hkv, a.tiles);
  if (nwq == 4) packed_dq_kernel<T, D, 4><<<nq, 256, 0, s>>>(a);
  else packed_dq_kernel<T, D, 1><<<nq, 64, 0, s>>>(a);
  if (a.Mk == 0) return;
  a.tiles = a.Mk / (32 * nwk) + a.B;
  a.d = deal(a.hkv, a.tiles);
  const unsigned nk = deal_grid(a.hkv, a.tiles);
  if (nwk == 4) packed_dkv_kernel<T, D, 4><<<nk, 256, 0, s>>>(a);
  else packed_dkv_kernel<T, D, 1><<<nk, 64, 0, s>>>(a);
}

}  // namespace ogv

using namespace ogv;

extern "C" size_t ogv_packed_attn_bwd_ws_bytes(const ogv_packed_desc* d, ogv_dtype dt) {
  if (packed_check("ogv_packed_attn_bwd_ws_bytes", d, dt) != OGV_OK) return 0;
  return (size_t)d->Mq * d->heads * sizeof(float);
}

extern "C" int ogv_packed_attn_bwd(const void* dout, const void* q, const void* k, const void* v, const void* out,
                                   const float* lse, const int* cu_q, const int* cu_k, void* dq, void* dk, void* dv,
                                   void* ws, const ogv_packed_desc* d, ogv_dtype dt, void* stream) {
  if (int rc = packed_check("ogv_packed_attn_bwd", d, dt)) return rc;
  OGV_REQUIRE(dout && q && out && lse && cu_q && cu_k && dq && ws && (d->Mk == 0 || (k && v && dk && dv)),
              "ogv_packed_attn_bwd: null pointer");
  OGV_REQUIRE(aligned16({dout, q, k, v, out, dq, dk, dv, ws}), "ogv_packed_attn_bwd: pointers must be 16-byte aligned");
  PackedArgs a;
  packed_args(d, a);
  a.q = q, a.k = k, a.v = v, a.o = out, a.dout = dout, a.lse = const_cast<float*>(lse), a.delta = (float*)ws;
  a.cu_q = cu_q, a.cu_k = cu_k, a.dq = dq, a.dk = dk, a.dv = dv;
  hipStream_t s = as_stream(stream);
#define OGV_BWD(T)                                   \
  if (d->D <= 32) bwd_launch<T, 32>(a, s);           \
  else if (d->D <= 64) bwd_launch<T, 64>(a, s);      \
  else if (d->D <= 96) bwd_launch<T, 96>(a, s);      \
  else bwd_launch<T, 128>(a, s);
  if (dt == OGV_BF16) { OGV_BWD(bf16) } else { OGV_BWD(float) }
#undef OGV_BWD
  return check_launch("ogv_packed_attn_bwd");
}
