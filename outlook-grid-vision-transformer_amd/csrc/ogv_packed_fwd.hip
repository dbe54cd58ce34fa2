// Attention over packed sequences of different lengths, forward.
//
//   s_rj = scale * q_r . k_j        key j of r's sequence, causal: j <= pos(r) + keys - queries
//   m_r = max_j s_rj,  l_r = sum_j exp(s_rj - m_r)
//   o_r = sum_j exp(s_rj - m_r) v_j / l_r,  lse_r = m_r + log(l_r);  no visible key: o_r = 0, lse_r = -inf
//
// One pass over the keys with a running maximum and sum.  A wave owns 32 rows; scores are computed
// transposed (S^T = K Q^T), so a row's scores lie in two lanes and its maximum, sum and rescaling are
// lane-local but for one exchange, and P^T feeds O^T += V^T P^T from registers.  K and V tiles pass
// through LDS once per workgroup.  Scores, maximum, sum and O are fp32; P is rounded to bf16 for the second
// product (a relative error of at most 2^-8 per weight, independent from key to key; the output's own rounding is as
// large).  For a backward, what rounding took from o is kept too (out_lo): see delta there.
//
// Split: four waves of 32 rows share the tiles (64 keys; 32 in fp32 and for one-wave workgroups of short sequences), two
// workgroups to a CU for D = 128, three for D = 64.  A row tile's keys are walked in one piece where there are row tiles
// enough for two to a CU; where there are fewer (single queries) they are cut into equal pieces whose partial results a
// second kernel joins.  The host decides by the numbers of rows, keys and sequences alone (the lengths are on the device):
// one long sequence among hundreds of short ones is walked by the waves that suit those, in one piece.
//
// What bounds it, measured on one MI355X (a large bf16 matrix product reaches 1365 TFLOP/s):
//   D = 128, causal, 16 heads on 4, sequences of 8191 and 5608: 405 to 411 us from box to box, 980 to 1000 TFLOP/s.  Left out
//     in turn (of 423 us then), the first product saved 117 us, the second 133, the copies to LDS 62, the exponentials 7: the
//     matrix instructions and the LDS reads that feed them (1 KB a product of 32 cycles, half the LDS rate from two waves a
//     SIMD) do not overlap further.
//   D = 64, 48 images of 196 to 1024 tokens, 12 heads: 92 to 95 us, 520 to 535 TFLOP/s.  29 us of it are the workgroups' ends
//     (q read, out written: 78 MB), the rest is spread over the 16-cycle exponentials (42 us for all of them with the other
//     vector instructions, by their count) and the latencies of 3 to 16 tiles a workgroup.
//   One query for each of 64 sequences (up to 8192 keys), 16 heads on 2: 30.7 us for 100 MB of keys and values, 3.3 TB/s, of
//     which the joining launch takes 5.
// The next tile's scores are computed before this tile's exponentials (466 -> 431 us at D = 128), copies bypass the
// registers (1318 -> 558), the reference of the weights moves lazily, heads are dealt evenly to the XCDs (558 -> 479).
#include "ogv_packed.h"

#include <initializer_list>

namespace ogv {

constexpr float LOG2E = 1.4426950408889634f;

// S^T = K Q^T of one key tile.
template <typename T, int D, int NB>
__device__ __forceinline__ void fwd_scores(const char* Ks, const Chunk (&qf)[Frag<T, D>::KK], f32x16 (&s)[NB], int lane) {
  constexpr int KK = Frag<T, D>::KK, RB = Frag<T, D>::RB;
  const int hf = lane >> 5, c = lane & 31;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    s[nb] = f32x16{};
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) mfma_step<T>(lds_chunk<RB>(Ks, nb * 32 + c, 2 * kk + hf), qf[kk], s[nb]);
  }
}

// Masks a tile's scores and moves the row's reference m (of the weights exp(scale (s - m))) where it has to; returns
// the exponent's offset.
template <int D, int NB>
__device__ __forceinline__ float fwd_reference(f32x16 (&s)[NB], f32x16 (&o)[D / 32], float& m, float& l, int key0, int lim, float c2,
                                               float grow, int hf) {
  if (!__all(key0 + NB * 32 - 1 <= lim)) {
    rare_branch();
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (key0 + nb * 32 + 8 * (i / 4) + 4 * hf + i % 4 > lim) s[nb][i] = -INFINITY;
  }
  float mx = s[0][0];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[nb][i]);
  mx = pair_max(mx);
  // The reference moves only where a row's maximum passed it by more than 2^8 (in weight): until then weights up to
  // 2^8 are as exact in fp32 and bf16 as those up to 1, and O need not be rescaled.  Each row decides for itself, so
  // its result does not depend on the rows beside it.
  if (__any(mx > m + grow)) {
    rare_branch();
    const float mn = mx > m + grow ? mx : m, mz = mn == -INFINITY ? 0.f : mn;
    const float corr = __builtin_amdgcn_exp2f((m - mz) * c2);
    m = mn;
    l *= corr;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[db][i] *= corr;
  }
  const float mz = m == -INFINITY ? 0.f : m;   // nothing visible yet: every weight is exp2(-inf) = 0
  const float mu = mz * c2;
  // exp2(s * c2 - mu) in one fma: the rounding of mu is the same factor in all weights taken against one reference, and
  // cancels among them.  When the reference moves, what was summed so far keeps the old one's: a relative 2^-24 |mu|,
  // which is what the scores themselves are off by.  Where mu is large, a row's reference is subtracted first.
  const bool far = fabsf(mu) > 16777216.f;
  if (__any(far)) {
    rare_branch();
    const float sub = far ? mz : 0.f;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[nb][i] -= sub;
    return far ? 0.f : mu;
  }
  return mu;
}

template <int NB> __device__ __forceinline__ void fwd_weights(f32x16 (&s)[NB], float& l, float c2, float mu) {
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float p = __builtin_amdgcn_exp2f(fmaf(s[nb][i], c2, -mu));
      s[nb][i] = p;
      l += p;
    }
}

// One row tile, which has rows, over keys kt0 * BN .. of its sequence.
template <typename T, int D, int NW, bool SPLIT>
__device__ __forceinline__ void fwd_rows(const PackedArgs& a, char* tiles, int h, const Seq& sq, int piece) {
  using F = Frag<T, D>;
  constexpr int BM = 32 * NW, BN = sizeof(T) == 2 && NW > 1 ? 64 : 32, NB = BN / 32;
  constexpr int KK = F::KK, E = F::E, TB = BN * F::RB;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hf = lane >> 5, c = lane & 31;
  const int b = sq.b, start = sq.start, len = sq.len, k0 = sq.start2, lk = sq.len2;
  const int rows = len * a.G, r0 = sq.tile * BM;
  // rows behind the last sequence belong to nothing: zeros
  const int store_rows = b == a.B - 1 ? (a.Mq - start) * a.G : rows;
  if (r0 >= store_rows) return;   // (never: but without it the compiler makes a slower split kernel, 31.2 us for 30.5)
  const int off = lk - len;
  int kend = r0 < rows ? lk : 0;
  if (a.causal && kend) kend = max(0, min(lk, group_div(min(r0 + BM, rows) - 1, a.G, a.gmagic) + off + 1));
  int kt0 = 0, kt1 = (kend + BN - 1) / BN, pieces = 1;
  if (SPLIT) {
    const int keys = piece_keys(lk, a.chunk, a.nsplit);
    pieces = max(1, (lk + keys - 1) / keys);
    kt0 = min(piece * (keys / BN), kt1);
    kt1 = min(kt0 + keys / BN, kt1);
  }

  const T* kb = (const T*)a.k + (long)k0 * a.rk + (long)h * a.hsk;
  const T* vb = (const T*)a.v + (long)k0 * a.rv + (long)h * a.hsv;
  TileCopy<T, D, BN, NW> kc, vc;
  kc.init(wave, lane, a.D, a.rk);
  vc.init(wave, lane, a.D, a.rv);
  // two K and two V tiles: while tile kt's weights are formed, tile kt + 1's scores are (its K is there) and K of
  // kt + 2 and V of kt + 1 are under way
  auto stage_k = [&](int kt, int at) { kc.load(kb + (long)kt * BN * a.rk, a.rk, lk - kt * BN, tiles + at, wave, lane, a.D); };
  auto stage_v = [&](int kt, int at) { vc.load(vb + (long)kt * BN * a.rv, a.rv, lk - kt * BN, tiles + 2 * TB + at, wave, lane, a.D); };
  if (kt0 < kt1) {
    stage_k(kt0, 0);
    stage_v(kt0, 0);
    if (kt0 + 1 < kt1) stage_k(kt0 + 1, TB);
  }

  const int r = r0 + wave * 32 + c, pos = group_div(r, a.G, a.gmagic), hg = r - pos * a.G;
  const bool live = r < rows;
  const int lim = live ? (a.causal ? min(lk - 1, pos + off) : lk - 1) : -1;   // last visible key
  Chunk qf[KK];
  {
    const T* qp = (const T*)a.q + (long)(start + (live ? pos : 0)) * a.rq + (long)(h * a.G + hg) * a.hsq;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const int d = (2 * kk + hf) * E;
      qf[kk] = zero_chunk();
      if (live && d < a.D) qf[kk].u = *reinterpret_cast<const uint4*>(qp + d);
    }
  }
  f32x16 o[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db) o[db] = f32x16{};
  float m = -INFINITY, l = 0.f;   // m: of q . k, before the scale; l: this lane's half of the row
  // (grow is finite, so that the first visible score always moves the reference from -inf, however small the scale)
  const float c2 = a.scale * LOG2E, grow = fminf(8.f / c2, 3e38f);

  if (kt0 < kt1) {
    f32x16 s[NB];
    tiles_ready();
    fwd_scores<T, D, NB>(tiles, qf, s, lane);
    int at = 0;
    for (int kt = kt0; kt + 1 < kt1; ++kt, at ^= TB) {
      const float mu = fwd_reference<D, NB>(s, o, m, l, kt * BN, lim, c2, grow, hf);
      tiles_ready();   // K of kt + 1, V of kt; and everybody is done with K of kt and V of kt - 1
      if (kt + 2 < kt1) stage_k(kt + 2, at);
      stage_v(kt + 1, at ^ TB);
      // the next scores' matrix instructions run under this tile's exponentials
      f32x16 next[NB];
      fwd_scores<T, D, NB>(tiles + (at ^ TB), qf, next, lane);
      fwd_weights<NB>(s, l, c2, mu);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) accum_xt<T, D>(tiles + 2 * TB + at, nb * 32, s[nb], o, lane);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) s[nb] = next[nb];
    }
    const float mu = fwd_reference<D, NB>(s, o, m, l, (kt1 - 1) * BN, lim, c2, grow, hf);
    tiles_ready();
    fwd_weights<NB>(s, l, c2, mu);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) accum_xt<T, D>(tiles + 2 * TB + at, nb * 32, s[nb], o, lane);
  }

  l = pair_sum(l);
  const bool out = r < store_rows;
  const long orow = (long)(start + pos) * a.hq + h * a.G + hg;   // row of the [Mq * hq] outputs
  if (SPLIT) {   // unnormalised partials, joined by packed_join_kernel
    const long at = (long)piece * a.Mq * a.hq + orow;
    store_cols<float, D>(a.part_o + at * a.D, o, 1.f, a.D, hf, out);
    if (out && hf == 0) {
      *reinterpret_cast<float2*>(a.part_ml + 2 * at) = make_float2(m, l);
      if (piece == 0) a.part_n[orow] = pieces;
    }
    return;
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);   // (NaN stays NaN)
  store_cols<T, D>((T*)a.out + (long)(start + pos) * a.ro + (long)(h * a.G + hg) * a.hso, o, inv, a.D, hf, out);
  if (sizeof(T) == 2 && a.out_lo) {
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = o[db][i] * inv;
        o[db][i] = x - (float)(T)x;
      }
    store_cols<T, D>((T*)a.out_lo + (long)(start + pos) * a.ro + (long)(h * a.G + hg) * a.hso, o, 1.f, a.D, hf, out);
  }
  if (out && hf == 0) a.lse[orow] = l == 0.f ? -INFINITY : m * a.scale + logf(l);
}

template <typename T, int D, int NW, bool SPLIT>
__global__ __launch_bounds__(NW * 64, sizeof(T) == 2 ? 2 : 1) void packed_fwd_kernel(const PackedArgs a) {
  constexpr int TB = (sizeof(T) == 2 && NW > 1 ? 64 : 32) * Frag<T, D>::RB;
  __shared__ __attribute__((aligned(16))) char tiles[4 * TB];
  const int lane = threadIdx.x & 63;
  if (a.D < D) clear_tiles<4 * TB, NW * 64>(tiles, threadIdx.x);
  if (SPLIT) {   // every piece of work, head by head
    for (int n = blockIdx.x;; n += gridDim.x) {
      Piece p;
      if (!find_piece(a, 32 * NW, n / a.hkv, lane, p)) return;
      fwd_rows<T, D, NW, true>(a, tiles, n % a.hkv, p.s, p.piece);
      __syncthreads();   // the tiles are free again
    }
  } else {
    int h, t;
    if (!head_tile(a.d, a.hkv, a.tiles, h, t)) return;
    Seq sq;
    if (!find_tile(a.cu_q, a.cu_k, a.B, a.Mq, a.Mk, a.G, 32 * NW, a.tiles - 1 - t, lane, sq)) return;
    fwd_rows<T, D, NW, false>(a, tiles, h, sq, 0);
  }
}

// out = sum_s w_s o_s / sum_s w_s l_s, w_s = exp(scale (m_s - max m)), over a row's key pieces in order.  A wave joins
// a row: lane s holds piece s's weight (at most 64), then the lanes are the dims.
template <typename T>
__global__ __launch_bounds__(256) void packed_join_kernel(const PackedArgs a) {
  const int lane = threadIdx.x & 63;
  const long R = (long)a.Mq * a.hq, row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= R) return;
  const int pieces = __builtin_amdgcn_readfirstlane(a.part_n[row]);
  float2 ml = make_float2(-INFINITY, 0.f);
  if (lane < a.nsplit) ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * (lane * R + row));
  if (lane >= pieces) ml = make_float2(-INFINITY, 0.f);   // (never written)
  const float m = group_max<64>(ml.x), mu = m == -INFINITY ? 0.f : m;
  float w = __builtin_amdgcn_exp2f((ml.x - mu) * (a.scale * LOG2E));
  const float l = wave_sum(w * ml.y);
  w *= l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);   // (NaN stays NaN)
  const int d = 2 * lane;
  float x = 0.f, y = 0.f;
  const float* po = a.part_o + row * a.D + (d < a.D ? d : 0);
  for (int s = 0; s < pieces; s += 4) {   // four loads under way; past the last piece it is repeated with weight 0
    float2 p[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) p[u] = *reinterpret_cast<const float2*>(po + min(s + u, pieces - 1) * R * a.D);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float ws = s + u < pieces ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), s + u)) : 0.f;
      x = fmaf(ws, p[u].x, x), y = fmaf(ws, p[u].y, y);
    }
  }
  const long q = row / a.hq;
  const float v[2] = {x, y};
  if (d < a.D) store_vec<T, 2>((T*)a.out + q * a.ro + (row - q * a.hq) * a.hso + d, v);
  if (sizeof(T) == 2 && a.out_lo) {
    const float lo[2] = {x - (float)(T)x, y - (float)(T)y};
    if (d < a.D) store_vec<T, 2>((T*)a.out_lo + q * a.ro + (row - q * a.hq) * a.hso + d, lo);
  }
  if (lane == 0) a.lse[row] = l == 0.f ? -INFINITY : m * a.scale + logf(l);
}

struct FwdPlan {
  int nw, tiles, nsplit, chunk;
  unsigned grid;
};

// Sequences that fill four waves' rows on average get them, others one wave per workgroup.  While there are fewer than
// 512 row tiles and at least two pieces of keys to a sequence on average, the keys are split into pieces of equal size (not
// equal number: sequences differ), about 800 in all (measured at one shape, 64 single queries, 97 thousand keys, 16 heads
// on 2 of 128: 30.8 us; 1024 pieces 31.5, 1500 32.9).
static FwdPlan fwd_plan(const ogv_packed_desc* d) {
  FwdPlan p;
  const long rows = (long)d->Mq * (d->heads / d->kv_heads);
  p.nw = rows >= 96L * d->B ? 4 : 1;
  p.tiles = (int)(rows / (32 * p.nw)) + d->B;
  const long blocks = (long)p.tiles * d->kv_heads;
  long chunk = ((long)d->Mk * blocks / d->B / 800 + 63) & ~63L;   // keys read by all row tiles over 800
  if (chunk < 128) chunk = 128;
  p.chunk = (int)(chunk < (1 << 30) ? chunk : 1 << 30);
  const bool split = blocks < 512 && d->Mk / d->B >= 2 * chunk;
  const long most = 4096 / (blocks > 0 ? blocks : 1);   // four times the average: bounds the workspace
  p.nsplit = !split ? 1 : (int)(most < 2 ? 2 : most > 64 ? 64 : most);
  long grid = blocks + (long)d->Mk / p.chunk * d->kv_heads * (p.tiles + d->B - 1) / d->B;
  p.grid = split ? (unsigned)(grid < 4096 ? grid : 4096) : deal_grid(d->kv_heads, p.tiles);
  return p;
}

template <typename T, int D>
static void fwd_launch(const FwdPlan& p, const PackedArgs& a, hipStream_t s) {
  if (p.nsplit > 1) {
    if (p.nw == 4) packed_fwd_kernel<T, D, 4, true><<<p.grid, 256, 0, s>>>(a);
    else packed_fwd_kernel<T, D, 1, true><<<p.grid, 64, 0, s>>>(a);
    packed_join_kernel<T><<<cdiv((long)a.Mq * a.hq, 4), 256, 0, s>>>(a);
  } else {
    if (p.nw == 4) packed_fwd_kernel<T, D, 4, false><<<p.grid, 256, 0, s>>>(a);
    else packed_fwd_kernel<T, D, 1, false><<<p.grid, 64, 0, s>>>(a);
  }
}

int packed_check(const char* what, const ogv_packed_desc* d, ogv_dtype dt) {
  OGV_REQUIRE(d, "%s: null descriptor", what);
  OGV_REQUIRE(dt == OGV_F32 || dt == OGV_BF16, "%s: bad dtype %d", what, (int)dt);
  OGV_REQUIRE(d->B > 0 && d->Mq > 0 && d->Mk >= 0, "%s: bad shape B=%d Mq=%d Mk=%d", what, d->B, d->Mq, d->Mk);
  OGV_REQUIRE(d->heads > 0 && d->kv_heads > 0 && d->heads % d->kv_heads == 0,
              "%s: heads=%d must be a multiple of kv_heads=%d", what, d->heads, d->kv_heads);
  OGV_REQUIRE(d->D >= 8 && d->D <= 128 && d->D % 8 == 0, "%s: head_dim=%d unsupported (need 8 <= D <= 128, D %% 8 == 0)",
              what, d->D);
  OGV_REQUIRE(d->scale > 0.f && __builtin_isfinite(d->scale), "%s: scale must be positive and finite", what);
  const long G = d->heads / d->kv_heads, most = 1L << 30;
  OGV_REQUIRE((long)d->Mq * G * G < 4 * most && (long)d->Mq * G < most && (long)d->Mk < most && d->B < most / 2,
              "%s: too many rows (Mq=%d, group %ld, Mk=%d)", what, d->Mq, G, d->Mk);
  const long grid = most * 2 - 8;
  OGV_REQUIRE(((long)d->Mq * G / 32 + d->B) * d->kv_heads < grid && ((long)d->Mk / 32 + d->B) * d->kv_heads < grid,
              "%s: grid too large", what);
  const long al = 16 / (dt == OGV_BF16 ? 2 : 4);
  for (int i = 0; i < OGV_PACKED_TENSORS; ++i) {
    // (offsets inside a tile of 64 rows, and between the heads of a group, are 32-bit)
    OGV_REQUIRE(G == 1 || (i != 0 && i != 4) || d->head[i] < (1L << 28) / G, "%s: head stride %d = %lld is too large", what, i,
                (long long)d->head[i]);
    OGV_REQUIRE(d->row[i] < (1 << 24), "%s: row stride %d = %lld is too large (below 2^24 elements)", what, i, (long long)d->row[i]);
    OGV_REQUIRE(d->row[i] >= 0 && d->head[i] >= 0 && d->row[i] % al == 0 && d->head[i] % al == 0,
                "%s: stride %d (row %lld, head %lld) must be non-negative multiples of 16 bytes", what, i,
                (long long)d->row[i], (long long)d->head[i]);
  }
  return OGV_OK;
}

void packed_args(const ogv_packed_desc* d, PackedArgs& a) {
  a = PackedArgs{};
  a.B = d->B, a.Mq = d->Mq, a.Mk = d->Mk, a.hq = d->heads, a.hkv = d->kv_heads, a.D = d->D;
  a.G = d->heads / d->kv_heads, a.causal = d->causal, a.scale = d->scale;
  a.gmagic = (unsigned)(((1ull << 32) + a.G - 1) / a.G);
  const int64_t *r = d->row, *h = d->head;
  a.rq = r[0], a.rk = r[1], a.rv = r[2], a.ro = r[3], a.rdo = r[4], a.rdq = r[5], a.rdk = r[6], a.rdv = r[7];
  a.hsq = h[0], a.hsk = h[1], a.hsv = h[2], a.hso = h[3], a.hsdo = h[4], a.hsdq = h[5], a.hsdk = h[6], a.hsdv = h[7];
}

bool aligned16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if ((uintptr_t)p & 15) return false;
  return true;
}

}  // namespace ogv

using namespace ogv;

extern "C" size_t ogv_packed_attn_fwd_ws_bytes(const ogv_packed_desc* d, ogv_dtype dt) {
  if (packed_check("ogv_packed_attn_fwd_ws_bytes", d, dt) != OGV_OK) return 0;
  const FwdPlan p = fwd_plan(d);
  return p.nsplit == 1 ? 0 : ((size_t)p.nsplit * (d->D + 2) + 1) * d->Mq * d->heads * sizeof(float);
}

extern "C" int ogv_packed_attn_fwd(const void* q, const void* k, const void* v, const int* cu_q, const int* cu_k,
                                   void* out, void* out_lo, float* lse, void* ws, const ogv_packed_desc* d, ogv_dtype dt,
                                   void* stream) {
  if (int rc = packed_check("ogv_packed_attn_fwd", d, dt)) return rc;
  OGV_REQUIRE(q && cu_q && cu_k && out && lse && (d->Mk == 0 || (k && v)), "ogv_packed_attn_fwd: null pointer");
  const FwdPlan p = fwd_plan(d);
  OGV_REQUIRE(p.nsplit == 1 || ws, "ogv_packed_attn_fwd: null workspace");
  OGV_REQUIRE(aligned16({q, k, v, out, out_lo, ws}), "ogv_packed_attn_fwd: pointers must be 16-byte aligned");
  PackedArgs a;
  packed_args(d, a);
  a.q = q, a.k = k, a.v = v, a.cu_q = cu_q, a.cu_k = cu_k, a.out = out, a.out_lo = out_lo, a.lse = lse;
  a.d = deal(d->kv_heads, p.tiles), a.tiles = p.tiles, a.nsplit = p.nsplit, a.chunk = p.chunk;
  const size_t n = (size_t)p.nsplit * d->Mq * d->heads;
  a.part_o = (float*)ws;
  a.part_ml = (float*)ws + n * d->D;
  a.part_n = (int*)((float*)ws + n * (d->D + 2));
  hipStream_t s = as_stream(stream);
#define OGV_FWD(T)                                      \
  if (d->D <= 32) fwd_launch<T, 32>(p, a, s);           \
  else if (d->D <= 64) fwd_launch<T, 64>(p, a, s);      \
  else if (d->D <= 96) fwd_launch<T, 96>(p, a, s);      \
  else fwd_launch<T, 128>(p, a, s);
  if (dt == OGV_BF16) { OGV_FWD(bf16) } else { OGV_FWD(float) }
#undef OGV_FWD
  return check_launch("ogv_packed_attn_fwd");
}
