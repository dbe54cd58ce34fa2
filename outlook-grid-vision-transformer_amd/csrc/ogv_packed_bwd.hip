// Attention over packed sequences, backward, from the forward's lse (probabilities are recomputed):
//
//   p_rj = exp(s_rj - lse_r)     delta_r = sum_d do_rd o_rd      dp_rj = do_r . v_j
//   ds_rj = p_rj (dp_rj - delta_r)
//   dq_r = scale sum_j ds_rj k_j      dk_j = scale sum_r ds_rj q_r      dv_j = sum_r p_rj do_r
//
// Two kernels, each owning the rows it writes, so no sum depends on the order of workgroups: dq walks the
// keys of a row block (and forms delta), dk / dv walk the rows -- of all query heads that share the key head --
// of a key block.  That computes the scores and dp twice (7 products for 5) and needs no atomics and no zeroed
// accumulators.  P and dS are rounded to bf16 for their products; scores, dp, delta and sums are fp32.  delta is taken
// from o and what its rounding left (out_lo): from the rounded o alone its error, common to a row's keys, was larger
// than dS's rounding (dq of short sequences: 0.0032 off in 2-norm instead of 0.0024).
//
// Measured on one MI355X: D = 128, causal, 16 heads on 4, sequences of 4096 and 2451 (327 GFLOP with the forward): dq 177 us
// (791 TFLOP/s of its three products), dk / dv 259 us (722, four products) and 23 us to add its row pieces.  Both are
// bound by the matrix instructions and the LDS reads that feed them (24 and 40 KB a 32x32 block of scores); dk / dv has all
// 256 registers of two waves a SIMD taken and 10 more in scratch.  D = 64, 64 images of 49 to 784 tokens, 6 heads: dq 55 us
// and dk / dv 58 us, of which 22 and 16 are the workgroups' ends (rows read and written); 5 tiles a workgroup do not hide the
// rest.  dq's keys are never split: with one query a sequence, its few waves walk all of them.
#include "ogv_packed.h"

#include <initializer_list>

namespace ogv {

int packed_check(const char* what, const ogv_packed_desc* d, ogv_dtype dt);
void packed_args(const ogv_packed_desc* d, PackedArgs& a);
bool aligned16(std::initializer_list<const void*> ps);

constexpr float BLOG2E = 1.4426950408889634f;

// 32 * NB keys of dq: scores and dp transposed (columns are rows r), dQ^T += K^T dS^T
template <typename T, int D, int NB>
__device__ __forceinline__ void dq_tile(const char* Ks, const char* Vs, const Chunk (&qf)[Frag<T, D>::KK],
                                        const Chunk (&gf)[Frag<T, D>::KK], f32x16 (&dq)[D / 32], int key0, int lim, float c2,
                                        float lse2, float delta, int lane) {
  constexpr int KK = Frag<T, D>::KK, RB = Frag<T, D>::RB;
  const int hf = lane >> 5, c = lane & 31;
  constexpr int AT_ONCE = D <= 64 ? NB : 1;   // larger heads have no registers for two blocks at once
#pragma unroll AT_ONCE
  for (int nb = 0; nb < NB; ++nb) {
    f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      mfma_step<T>(lds_chunk<RB>(Ks, nb * 32 + c, 2 * kk + hf), qf[kk], s);
      mfma_step<T>(lds_chunk<RB>(Vs, nb * 32 + c, 2 * kk + hf), gf[kk], dp);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c2, -lse2)) * (dp[i] - delta);
    if (!__all(key0 + nb * 32 + 31 <= lim)) {
      rare_branch();
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (key0 + nb * 32 + 8 * (i / 4) + 4 * hf + i % 4 > lim) s[i] = 0.f;
    }
    accum_xt<T, D>(Ks, nb * 32, s, dq, lane);
  }
}

template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64, sizeof(T) == 2 ? 2 : 1) void packed_dq_kernel(const PackedArgs a) {
  using F = Frag<T, D>;
  constexpr int BM = 32 * NW, BN = sizeof(T) == 2 && NW > 1 ? 64 : 32, NB = BN / 32;
  constexpr int RB = F::RB, KK = F::KK, E = F::E, TB = BN * RB;
  __shared__ __attribute__((aligned(16))) char tiles[4 * TB];   // K and V, two of each
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hf = lane >> 5, c = lane & 31;

  int h, t;
  if (!head_tile(a.d, a.hkv, a.tiles, h, t)) return;
  if (a.D < D) clear_tiles<4 * TB, NW * 64>(tiles, tid);
  Seq sq;
  if (!find_tile(a.cu_q, a.cu_k, a.B, a.Mq, a.Mk, a.G, BM, a.tiles - 1 - t, lane, sq)) return;
  const int k0 = sq.start2, lk = sq.len2;
  const int rows = sq.len * a.G, r0 = sq.tile * BM;
  const int store_rows = sq.b == a.B - 1 ? (a.Mq - sq.start) * a.G : rows;
  const int off = lk - sq.len;
  int kend = r0 < rows ? lk : 0;
  if (a.causal && kend) kend = max(0, min(lk, group_div(min(r0 + BM, rows) - 1, a.G, a.gmagic) + off + 1));
  const int kt1 = (kend + BN - 1) / BN;

  const T* kb = (const T*)a.k + (long)k0 * a.rk + (long)h * a.hsk;
  const T* vb = (const T*)a.v + (long)k0 * a.rv + (long)h * a.hsv;
  TileCopy<T, D, BN, NW> kc, vc;
  kc.init(wave, lane, a.D, a.rk);
  vc.init(wave, lane, a.D, a.rv);
  auto stage = [&](int kt, int at) {
    kc.load(kb + (long)kt * BN * a.rk, a.rk, lk - kt * BN, tiles + at, wave, lane, a.D);
    vc.load(vb + (long)kt * BN * a.rv, a.rv, lk - kt * BN, tiles + at + TB, wave, lane, a.D);
  };
  if (kt1 > 0) stage(0, 0);

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
        Chunk oc, lc = zero_chunk();
        oc.u = *reinterpret_cast<const uint4*>(op + d);
        if constexpr (sizeof(T) == 2) {
          if (a.o_lo) lc.u = *reinterpret_cast<const uint4*>((const T*)a.o_lo + row * a.ro + head * a.hso + d);
#pragma unroll
          for (int e = 0; e < 8; ++e) delta = fmaf((float)gf[kk].h[e], (float)oc.h[e] + (float)lc.h[e], delta);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) delta = fmaf(gf[kk].f[e], oc.f[e], delta);
        }
      }
    }
  }
  delta = pair_sum(delta);
  // a row that sees nothing has lse = -inf: +inf keeps its weights at exp2(-inf) = 0
  float lse2 = live ? a.lse[orow] * BLOG2E : INFINITY;
  if (lse2 == -INFINITY) lse2 = INFINITY;
  if (live && hf == 0) a.rowstat[orow] = make_float2(lse2, delta);   // for the dk / dv kernel
  f32x16 dq[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db) dq[db] = f32x16{};
  const float c2 = a.scale * BLOG2E;

  for (int kt = 0, at = 0; kt < kt1; ++kt, at ^= 2 * TB) {
    tiles_ready();
    if (kt + 1 < kt1) stage(kt + 1, at ^ (2 * TB));
    dq_tile<T, D, NB>(tiles + at, tiles + at + TB, qf, gf, dq, kt * BN, lim, c2, lse2, delta, lane);
  }

  store_cols<T, D>((T*)a.dq + (long)(sq.start + pos) * a.rdq + (long)(h * a.G + hg) * a.hsdq, dq, a.scale, a.D, hf, r < store_rows);
}

// 32 * NB rows of dk / dv: scores and dp with columns = keys, dV^T += dO^T P, dK^T += Q^T dS.  With V in LDS (VL) nearly all
// registers are taken and the compiler would put each LDS read right before its product; read one product ahead instead
// (long causal streams, D = 128: the step 555 -> 535 us; heads of 64, and dq, have the registers and gain nothing).
template <typename T, int D, int NB, bool VL>
__device__ __forceinline__ void dkv_tile(const char* Qs, const char* Gs, const float2* St, const Chunk (&kf)[Frag<T, D>::KK],
                                         const Chunk (&vf)[VL ? 1 : Frag<T, D>::KK], const char* Vs, f32x16 (&dk)[D / 32], f32x16 (&dv)[D / 32], int rt,
                                         int off, int j, int jmax, const PackedArgs& a, float c2, int lane) {
  constexpr int KK = Frag<T, D>::KK, RB = Frag<T, D>::RB;
  const int hf = lane >> 5, c = lane & 31;
  constexpr int AT_ONCE = D <= 64 ? NB : 1;   // larger heads have no registers for two blocks at once
#pragma unroll AT_ONCE
  for (int nb = 0; nb < NB; ++nb) {
    f32x16 s = f32x16{}, dp = f32x16{};
    Chunk qa = lds_chunk<RB>(Qs, nb * 32 + c, hf), ga = lds_chunk<RB>(Gs, nb * 32 + c, hf), va;
    if (VL) va = lds_chunk<RB>(Vs, c, hf);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const int nx = 2 * (kk + 1) + hf;
      Chunk qn = qa, gn = ga, vn = va;
      if (kk + 1 < KK) {
        qn = lds_chunk<RB>(Qs, nb * 32 + c, nx), gn = lds_chunk<RB>(Gs, nb * 32 + c, nx);
        if (VL) vn = lds_chunk<RB>(Vs, c, nx);
      }
      if (VL) __builtin_amdgcn_sched_barrier(0);
      mfma_step<T>(qa, kf[kk], s);
      mfma_step<T>(ga, VL ? va : vf[VL ? 0 : kk], dp);
      if (VL) __builtin_amdgcn_sched_barrier(0);
      qa = qn, ga = gn, va = vn;
    }
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const f32x4 st = *reinterpret_cast<const f32x4*>(St + nb * 32 + 8 * (i / 4) + 4 * hf + i % 4);   // lse, delta of two rows
      s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c2, -st[0]));
      s[i + 1] = __builtin_amdgcn_exp2f(fmaf(s[i + 1], c2, -st[2]));
      dp[i] -= st[1];
      dp[i + 1] -= st[3];
    }
    const int r0 = rt + nb * 32;
    if (a.causal && group_div(r0, a.G, a.gmagic) + off < jmax) {   // (the first row of the block sees least)
      rare_branch();
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (j > group_div(r0 + 8 * (i / 4) + 4 * hf + i % 4, a.G, a.gmagic) + off) s[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) dp[i] *= s[i];
    accum_xt<T, D, VL>(Gs, nb * 32, s, dv, lane);
    accum_xt<T, D, VL>(Qs, nb * 32, dp, dk, lane);
  }
}

// A workgroup owns 32 * NW keys (32 per wave, K and the sums in registers) and one of a.nsplit pieces of the rows
// that see them.  Heads of 96 and 128 keep V in LDS instead of registers: that leaves two waves to a SIMD (at one,
// nothing covers the exponentials and the LDS reads).  One piece writes dk, dv; several write fp32 partial sums.
template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64, sizeof(T) == 2 && (NW > 1 || D < 128) ? 2 : 1) void packed_dkv_kernel(const PackedArgs a) {
  using F = Frag<T, D>;
  constexpr bool VL = sizeof(T) == 2 && D >= 96;
  constexpr int BM = 32 * NW, BN = sizeof(T) == 2 && NW > 1 && !VL ? 64 : 32, NB = BN / 32;   // BM keys, BN rows per step
  constexpr int RB = F::RB, KK = F::KK, E = F::E, NT = 64 * NW, TB = BN * RB;
  // (a step of 32 rows of a 96-wide head is one and a half instructions of four waves: the last half is left out)
  constexpr int NI = (BN * F::NC + NT - 1) / NT;
  __shared__ __attribute__((aligned(16))) char tiles[4 * TB];   // q and dout, two of each
  __shared__ __attribute__((aligned(16))) char Vl[VL ? BM * RB : 16];
  __shared__ __attribute__((aligned(16))) float2 stats[2 * BN];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hf = lane >> 5, c = lane & 31;

  int h, t;
  if (!head_tile(a.d, a.hkv, a.tiles * a.nsplit, h, t)) return;
  if (a.D < D) clear_tiles<4 * TB, NT>(tiles, tid);
  if (VL && a.D < D) clear_tiles<sizeof(Vl), NT>(Vl, tid);
  const int split = t % a.nsplit;
  Seq sk;
  if (!find_tile(a.cu_k, a.cu_q, a.B, a.Mk, a.Mq, 1, BM, t / a.nsplit, lane, sk)) return;
  const int q0 = sk.start2, lq = sk.len2;
  const int j0 = sk.tile * BM, off = sk.len - lq, rows = lq * a.G;
  const int store_keys = sk.b == a.B - 1 ? a.Mk - sk.start : sk.len;
  int rend = j0 < sk.len ? rows : 0, rbeg = 0;
  if (a.causal) rbeg = (int)(min((long)rend, (long)max(0, j0 - off) * a.G) / BN) * BN;   // rows that see key j0 or later
  if (a.nsplit > 1) {
    const int per = ((rend - rbeg + a.nsplit - 1) / a.nsplit + BN - 1) / BN * BN;
    rbeg = min(rbeg + split * per, rend);
    rend = min(rbeg + per, rend);
  }

  const T* qb = (const T*)a.q + (long)q0 * a.rq + (long)h * a.G * a.hsq;
  const T* gb = (const T*)a.dout + (long)q0 * a.rdo + (long)h * a.G * a.hsdo;
  const float2* sb = a.rowstat + (long)q0 * a.hq + h * a.G;
  float2 st = make_float2(0.f, 0.f);
  // byte offsets of a lane's chunks from row rt's query, for rr = rt + row clamped by the caller
  auto place = [&](int n, int rt, int p0, int last, unsigned& oq, unsigned& og) {
    const int slot = (n * NW + wave) * 64 + lane, row = slot / F::NC, ch = (slot - row * F::NC) ^ swz<RB>(row);
    const int rr = min(rt + row, last), pos = group_div(rr, a.G, a.gmagic);
    const unsigned hg = (unsigned)(rr - pos * a.G), dp = (unsigned)(pos - p0), col = ch * 16;
    oq = dp * (unsigned)(a.rq * sizeof(T)) + hg * (unsigned)(a.hsq * sizeof(T)) + col;
    og = dp * (unsigned)(a.rdo * sizeof(T)) + hg * (unsigned)(a.hsdo * sizeof(T)) + col;
    if (ch * E >= a.D) oq = NO_CHUNK;
  };
  unsigned oq[NI], og[NI];   // of a whole step whose first row is its query's first head (always, where G divides BN)
#pragma unroll
  for (int n = 0; n < NI; ++n) place(n, 0, 0, BN, oq[n], og[n]);
  const bool even = BN % a.G == 0;
  // rows rt .. rt + BN - 1 (the last one repeated) of q and dout to LDS; their statistics to registers
  auto stage = [&](int rt, int at) {
    const int p0 = group_div(rt, a.G, a.gmagic);
    const char* qt = uniform_ptr(qb + (long)p0 * a.rq);
    const char* gt = uniform_ptr(gb + (long)p0 * a.rdo);
    const bool whole = even && rt + BN <= rows;
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      if (BN * F::NC % NT != 0 && (n * NW + wave) * 64 >= BN * F::NC) break;   // (uniform in a wave)
      unsigned x = oq[n], y = og[n];
      if (!whole) place(n, rt, p0, rows - 1, x, y);
      if (a.D == D || x != NO_CHUNK) {
        copy16(qt, x, tiles + at + (n * NW + wave) * 1024);
        copy16(gt, y, tiles + at + TB + (n * NW + wave) * 1024);
      }
    }
    if (tid < BN) {
      const int rr = min(rt + tid, rows - 1), pos = group_div(rr, a.G, a.gmagic);
      st = sb[(long)pos * a.hq + (rr - pos * a.G)];
      if (rt + tid >= rows) st = make_float2(INFINITY, 0.f);   // no such row: weight 0
    }
  };
  const int j = j0 + wave * 32 + c, jmax = j0 + wave * 32 + 31;
  const bool live = j < sk.len;
  Chunk kf[KK], vf[VL ? 1 : KK];
  if (rbeg < rend) {
    stage(rbeg, 0);
    if constexpr (VL) {
      TileCopy<T, D, BM, NW> vc;
      vc.init(wave, lane, a.D, a.rv);
      vc.load((const T*)a.v + (long)(sk.start + j0) * a.rv + (long)h * a.hsv, a.rv, sk.len - j0, Vl, wave, lane, a.D);
    }
    const T* kp = (const T*)a.k + (long)(sk.start + (live ? j : j0)) * a.rk + (long)h * a.hsk;
    const T* vp = (const T*)a.v + (long)(sk.start + (live ? j : j0)) * a.rv + (long)h * a.hsv;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const int d = (2 * kk + hf) * E;
      kf[kk] = zero_chunk();
      if (d < a.D) kf[kk].u = *reinterpret_cast<const uint4*>(kp + d);
      if constexpr (!VL) {
        vf[kk] = zero_chunk();
        if (d < a.D) vf[kk].u = *reinterpret_cast<const uint4*>(vp + d);
      }
    }
  }
  f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db) dk[db] = f32x16{}, dv[db] = f32x16{};
  const float c2 = a.scale * BLOG2E;
  const char* Vw = Vl + (VL ? wave * 32 * RB : 0);

  for (int rt = rbeg, at = 0; rt < rend; rt += BN, at ^= 2 * TB) {
    float2* S = stats + (at ? BN : 0);
    if (tid < BN) S[tid] = st;
    tiles_ready();
    if (rt + BN < rend) stage(rt + BN, at ^ (2 * TB));
    dkv_tile<T, D, NB, VL>(tiles + at, tiles + at + TB, S, kf, vf, Vw, dk, dv, rt, off, j, jmax, a, c2, lane);
  }

  const bool out = j < store_keys;
  if (!live) {   // keys behind the last sequence
#pragma unroll
    for (int db = 0; db < D / 32; ++db) dk[db] = f32x16{}, dv[db] = f32x16{};
  }
  if (a.nsplit > 1) {
    const long n = (long)a.Mk * a.hkv, row = (long)(sk.start + j) * a.hkv + h;
    store_cols<float, D>(a.part_o + ((2L * split) * n + row) * a.D, dk, 1.f, a.D, hf, out);
    store_cols<float, D>(a.part_o + ((2L * split + 1) * n + row) * a.D, dv, 1.f, a.D, hf, out);
    return;
  }
  store_cols<T, D>((T*)a.dk + (long)(sk.start + j) * a.rdk + (long)h * a.hsdk, dk, a.scale, a.D, hf, out);
  store_cols<T, D>((T*)a.dv + (long)(sk.start + j) * a.rdv + (long)h * a.hsdv, dv, 1.f, a.D, hf, out);
}

// dk, dv = sums of the row pieces, in order
template <typename T>
__global__ __launch_bounds__(256) void packed_sum_kernel(const PackedArgs a) {
  const int per = a.D / 4;
  const long n = (long)a.Mk * a.hkv, idx = (long)blockIdx.x * 256 + threadIdx.x;
  if (idx >= 2 * n * per) return;
  const long row2 = idx / per, row = row2 >> 1, key = row / a.hkv;   // dk and dv of a row next to each other
  const int d = (int)(idx - row2 * per) * 4, which = (int)(row2 & 1), h = (int)(row - key * a.hkv);
  float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < a.nsplit; ++s) {
    const float4 p = *reinterpret_cast<const float4*>(a.part_o + ((2L * s + which) * n + row) * a.D + d);
    x[0] += p.x, x[1] += p.y, x[2] += p.z, x[3] += p.w;
  }
  const float mul = which ? 1.f : a.scale;
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] *= mul;
  T* out = which ? (T*)a.dv + key * a.rdv + h * a.hsdv : (T*)a.dk + key * a.rdk + h * a.hsdk;
  store_vec<T, 4>(out + d, x);
}

struct BwdPlan {
  int nwq, nwk, tiles_q, tiles_k, nsplit;
};

// Waves per workgroup as in the forward.  The rows of dk / dv are split while the key tiles would not fill the 256 CUs
// twice, into 1024 workgroups or a few more (two to a CU, twice: under the causal mask the first tile has twice the
// average work; measured on long causal streams, D = 128, alone: with 768 the step takes 1.06, with 1536 1.04 times as long).  A piece costs
// 16 bytes of partial sums per key, head and dim, so it has at least 512 rows on average, 32 in fp32, whose products run
// at a sixteenth of the rate.
static BwdPlan bwd_plan(const ogv_packed_desc* d, ogv_dtype dt) {
  BwdPlan p;
  const long rows = (long)d->Mq * (d->heads / d->kv_heads);
  p.nwq = rows >= 96L * d->B ? 4 : 1, p.nwk = d->Mk >= 96L * d->B ? 4 : 1;
  p.tiles_q = (int)(rows / (32 * p.nwq)) + d->B;
  p.tiles_k = d->Mk / (32 * p.nwk) + d->B;
  const long blocks = (long)p.tiles_k * d->kv_heads;
  long n = blocks < 512 ? (1024 + blocks - 1) / blocks : 1;
  const long most = rows / d->B / (dt == OGV_BF16 ? 512 : 32);
  if (n > most) n = most;
  p.nsplit = (int)(n < 1 ? 1 : n > 16 ? 16 : n);
  return p;
}

template <typename T, int D>
static void bwd_launch(const BwdPlan& p, PackedArgs a, hipStream_t s) {
  a.tiles = p.tiles_q, a.d = deal(a.hkv, a.tiles);
  const unsigned nq = deal_grid(a.hkv, a.tiles);
  if (p.nwq == 4) packed_dq_kernel<T, D, 4><<<nq, 256, 0, s>>>(a);
  else packed_dq_kernel<T, D, 1><<<nq, 64, 0, s>>>(a);
  if (a.Mk == 0) return;
  a.tiles = p.tiles_k, a.nsplit = p.nsplit, a.d = deal(a.hkv, a.tiles * a.nsplit);
  const unsigned nk = deal_grid(a.hkv, a.tiles * a.nsplit);
  if (p.nwk == 4) packed_dkv_kernel<T, D, 4><<<nk, 256, 0, s>>>(a);
  else packed_dkv_kernel<T, D, 1><<<nk, 64, 0, s>>>(a);
  if (a.nsplit > 1) packed_sum_kernel<T><<<cdiv((long)a.Mk * a.hkv * (a.D / 2), 256), 256, 0, s>>>(a);
}

}  // namespace ogv

using namespace ogv;

extern "C" size_t ogv_packed_attn_bwd_ws_bytes(const ogv_packed_desc* d, ogv_dtype dt) {
  if (packed_check("ogv_packed_attn_bwd_ws_bytes", d, dt) != OGV_OK) return 0;
  const BwdPlan p = bwd_plan(d, dt);
  const size_t stat = ((size_t)d->Mq * d->heads * 2 + 3) & ~(size_t)3;
  return (stat + (p.nsplit > 1 ? (size_t)p.nsplit * 2 * d->Mk * d->kv_heads * d->D : 0)) * sizeof(float);
}

extern "C" int ogv_packed_attn_bwd(const void* dout, const void* q, const void* k, const void* v, const void* out, const void* out_lo,
                                   const float* lse, const int* cu_q, const int* cu_k, void* dq, void* dk, void* dv,
                                   void* ws, const ogv_packed_desc* d, ogv_dtype dt, void* stream) {
  if (int rc = packed_check("ogv_packed_attn_bwd", d, dt)) return rc;
  OGV_REQUIRE(dout && q && out && lse && cu_q && cu_k && dq && ws && (d->Mk == 0 || (k && v && dk && dv)),
              "ogv_packed_attn_bwd: null pointer");
  OGV_REQUIRE(aligned16({dout, q, k, v, out, out_lo, dq, dk, dv, ws}), "ogv_packed_attn_bwd: pointers must be 16-byte aligned");
  PackedArgs a;
  packed_args(d, a);
  a.q = q, a.k = k, a.v = v, a.o = out, a.o_lo = out_lo, a.dout = dout, a.lse = const_cast<float*>(lse), a.rowstat = (float2*)ws;
  a.cu_q = cu_q, a.cu_k = cu_k, a.dq = dq, a.dk = dk, a.dv = dv;
  a.part_o = (float*)ws + (((size_t)d->Mq * d->heads * 2 + 3) & ~(size_t)3);
  const BwdPlan p = bwd_plan(d, dt);
  hipStream_t s = as_stream(stream);
#define OGV_BWD(T)                                      \
  if (d->D <= 32) bwd_launch<T, 32>(p, a, s);           \
  else if (d->D <= 64) bwd_launch<T, 64>(p, a, s);      \
  else if (d->D <= 96) bwd_launch<T, 96>(p, a, s);      \
  else bwd_launch<T, 128>(p, a, s);
  if (dt == OGV_BF16) { OGV_BWD(bf16) } else { OGV_BWD(float) }
#undef OGV_BWD
  return check_launch("ogv_packed_attn_bwd");
}
