// Shared pieces of the packed-sequence attention kernels (ogv_packed_fwd.hip, ogv_packed_bwd.hip).
//
// Rows.  The G = heads / kv_heads query heads that share a key / value head are extra rows of one
// problem: row r of sequence b and key / value head h is query r / G, head h * G + r % G.  A key /
// value tile is then read once for the whole group, and a single query still fills G rows.
//
// Fragments (32x32 MFMA, lane = 32 * hf + c, hf = lane >> 5, c = lane & 31; a 16-B chunk holds E = 8
// bf16 or 4 fp32 values):
//   A / B operand of reduction step kk: row (column) c, chunk 2 * kk + hf.  bf16: one 32x32x16 product.
//     fp32: four 32x32x2 products, element e of the chunk each.  Both operands are read alike, so the
//     order of the reduction inside a step does not matter.
//   C / D: column c, rows 8 * (i / 4) + 4 * hf + i % 4 in register i = 0..15.
//   A C tile is the B operand of the next product as it stands: register 8 * s + j (bf16) goes to
//   reduction slot j, so the A operand takes rows 16 * s + 4 * hf + {0..3} and + 8 -- what two
//   ds_read_b64_tr_b16 of a row-major LDS tile deliver -- and for fp32 register i is one product with
//   row 8 * (i / 4) + 4 * hf + i % 4.
//
// LDS tiles are row-major without padding; 16-B chunk ch of row r sits at ch ^ swz(r).  With RB bytes a
// row, swz keeps both access shapes free of bank conflicts: 16 rows of one chunk (b128 operand reads) and
// 4 rows of 64 B (transposed reads).
#pragma once
#include "ogv_common.h"
#include "ogv_packed_tiles.h"

namespace ogv {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((address_space(3))) s16x4 lds_tr_t;

// Workgroup -> (key / value head, tile slot).  Each head is dealt to as few XCDs as an even share allows, tile slots
// alternating between them: the workgroups of an XCD walk the same keys (its L2 holds them) and every XCD gets
// the same mix of early and late tiles, which differ in work under the causal mask.
struct Deal {
  int parts;   // interleaved parts of a head
  int per;     // tile slots of a part
};
static inline Deal deal(int hkv, int tiles) {
  int g = 8;
  while (hkv % g) g >>= 1;
  const int parts = 8 / g;
  return Deal{parts, (tiles + parts - 1) / parts};
}
static inline unsigned deal_grid(int hkv, int tiles) {
  const Deal d = deal(hkv, tiles);
  return (unsigned)((long)hkv * d.parts * d.per);
}
__device__ __forceinline__ bool head_tile(const Deal d, int hkv, int tiles, int& h, int& t) {
  const int x = blockIdx.x & 7, y = blockIdx.x >> 3, mine = hkv * d.parts / 8;
  const int part = x * mine + y / d.per;
  h = part / d.parts;
  t = (y % d.per) * d.parts + part % d.parts;
  return t < tiles;
}

struct PackedArgs {
  const void *q, *k, *v, *o, *o_lo, *dout;   // o, o_lo: forward's outputs (read by the backward)
  void *out, *out_lo, *dq, *dk, *dv;
  float* lse;
  float2* rowstat;                    // backward: lse * log2(e) (+inf where no key is seen) and delta of a row
  const int *cu_q, *cu_k;
  float *part_o, *part_ml;            // split forward: [piece][Mq * hq][D] and [piece][Mq * hq][2]
  int* part_n;                        // split forward: pieces of a row
  int B, Mq, Mk, hq, hkv, D, G, causal;
  unsigned gmagic;                    // ceil(2^32 / G); r / G = umulhi(r, gmagic) for r * G < 2^32
  Deal d;                             // workgroups of the unsplit kernels
  int tiles, nsplit, chunk;           // tile slots per key / value head; most key pieces of a row, fewest keys of a piece
  float scale;
  long rq, rk, rv, ro, rdo, rdq, rdk, rdv;   // row strides, elements
  long hsq, hsk, hsv, hso, hsdo, hsdq, hsdk, hsdv;   // head strides, elements
};

// r / G (G == 1 has no 32-bit magic number)
__device__ __forceinline__ int group_div(int r, int G, unsigned magic) {
  return G == 1 ? r : (int)__umulhi((unsigned)r, magic);
}

template <int RB> __device__ __forceinline__ int swz(int r) {
  if constexpr (RB % 256 == 0) return ((r & 3) << 2) | ((r >> 2) & 3);
  else if constexpr (RB % 128 == 0) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
  else return (r >> 2) & 3;
}

template <typename T, int D> struct Frag {
  static constexpr int E = 16 / sizeof(T);          // elements per 16-B chunk
  static constexpr int RB = D * (int)sizeof(T);     // bytes per LDS row
  static constexpr int NC = RB / 16;                // chunks per row
  static constexpr int KK = NC / 2;                 // reduction steps over D
};

union Chunk {
  uint4 u;
  bf16x8 h;
  f32x4 f;
};

// a: this lane's of lanes 0..31 and its partner's (lane ^ 32) of lanes 32..63 afterwards stand where the MFMA layout
// has halves apart: (a, b) -> ({a of the lower half, b of the lower half}, {a of the upper half, b of the upper half})
__device__ __forceinline__ void swap_halves(unsigned& a, unsigned& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0], b = r[1];
}
// the larger of a value and its partner's in lane ^ 32
__device__ __forceinline__ float pair_max(float v) {
  unsigned a = __builtin_bit_cast(unsigned, v), b = a;
  swap_halves(a, b);
  return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ __forceinline__ float pair_sum(float v) {
  unsigned a = __builtin_bit_cast(unsigned, v), b = a;
  swap_halves(a, b);
  return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}

__device__ __forceinline__ Chunk zero_chunk() {
  Chunk c;
  c.u = make_uint4(0, 0, 0, 0);
  return c;
}

// acc += A . B over one reduction step
template <typename T> __device__ __forceinline__ void mfma_step(const Chunk& a, const Chunk& b, f32x16& acc) {
  if constexpr (sizeof(T) == 2) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.h, b.h, acc, 0, 0, 0);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.f[e], b.f[e], acc, 0, 0, 0);
  }
}

template <int RB> __device__ __forceinline__ Chunk lds_chunk(const char* tile, int row, int ch) {
  Chunk c;
  c.u = *reinterpret_cast<const uint4*>(tile + row * RB + ((ch ^ swz<RB>(row)) << 4));
  return c;
}

// 16 bytes a lane, from base + off (base uniform) straight to LDS: lane i's to l + 16 * i.  In assembly because the
// compiler would make every later LDS read wait for the copy, whichever tile it writes; nothing comes back in registers,
// and tiles_ready() below waits before anybody reads the tile.  m0 holds the LDS address; its write needs a wait state.  m0
// is named as clobbered, so that no write of it by the compiler, for an instruction of its own, is taken to live past the
// copy (the compiler reserves m0 and warns about that: switched off).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void copy16(const char* base, unsigned off, char* l) {
  const unsigned at = (unsigned)(uint64_t)l;   // an LDS address is the low half of its generic one
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(at)), "v"(off),
               "s"(base)
               : "memory", "m0");
}
#pragma clang diagnostic pop

template <typename P> __device__ __forceinline__ const char* uniform_ptr(const P* p) {
  const uint64_t v = (uint64_t)p;
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)v), hi = __builtin_amdgcn_readfirstlane((unsigned)(v >> 32));
  return reinterpret_cast<const char*>(((uint64_t)hi << 32) | lo);
}

constexpr unsigned NO_CHUNK = ~0u;   // a chunk past the head: not copied, its place in the tile holds zeros (clear_tiles)

// Copies ROWS rows of a strided tensor into an LDS tile, straight from global memory to LDS (no registers): one
// instruction of a wave fills 64 consecutive chunks, so the swizzle is in the addresses that the lanes read.  Rows past
// the last one repeat it: whoever uses the tile masks their products.  Offsets inside a tile are 32-bit (row strides are
// below 2^24 elements), the tile's base is a uniform pointer.
template <typename T, int D, int ROWS, int NW> struct TileCopy {
  using F = Frag<T, D>;
  static constexpr int NI = ROWS * F::NC / (64 * NW);
  static_assert(ROWS * F::NC % (64 * NW) == 0, "whole instructions");
  unsigned off[NI];   // of this lane's chunks: row * stride + chunk, bytes
  static __device__ __forceinline__ unsigned place(int slot, int last, int Dlive, long stride) {
    const int row = slot / F::NC, ch = (slot - row * F::NC) ^ swz<F::RB>(row);
    return ch * F::E < Dlive ? (unsigned)min(row, last) * (unsigned)(stride * sizeof(T)) + ch * 16 : NO_CHUNK;
  }
  __device__ __forceinline__ void init(int wave, int lane, int Dlive, long stride) {
#pragma unroll
    for (int n = 0; n < NI; ++n) off[n] = place((n * NW + wave) * 64 + lane, ROWS, Dlive, stride);
  }
  // rows 0 .. ROWS - 1 behind base, of which `left` >= 1 exist
  __device__ __forceinline__ void load(const T* base, long stride, int left, char* tile, int wave, int lane, int Dlive) const {
    const char* b = uniform_ptr(base);
    if (left >= ROWS && Dlive == D) {
#pragma unroll
      for (int n = 0; n < NI; ++n) copy16(b, off[n], tile + (n * NW + wave) * 1024);
    } else {
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        const unsigned at = left >= ROWS ? off[n] : place((n * NW + wave) * 64 + lane, left - 1, Dlive, stride);
        if (at != NO_CHUNK) copy16(b, at, tile + (n * NW + wave) * 1024);
      }
    }
  }
};

// Zeros for the chunks that no copy writes; once, before the first copy.
template <int BYTES, int NT> __device__ __forceinline__ void clear_tiles(char* tiles, int tid) {
  for (int i = tid; i < BYTES / 16; i += NT) reinterpret_cast<uint4*>(tiles)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
}

// Keeps the compiler from running a wave-uniform branch's body always and selecting its results.
__device__ __forceinline__ void rare_branch() { asm volatile(""); }

// This wave's copies to LDS are done; then everybody's are.
__device__ __forceinline__ void tiles_ready() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// B operand of the next product: 16 rows (bf16) of a C tile, registers 8 * s .. 8 * s + 7
__device__ __forceinline__ Chunk pack8(const f32x16& x, int s) {
  Chunk c;
#pragma unroll
  for (int j = 0; j < 8; ++j) c.h[j] = (bf16)x[8 * s + j];
  return c;
}

// acc[db] += X^T . Y for one 32-row block of the LDS tile: X is rows row0 .. row0 + 31 of the tile, y the
// C tile whose rows are the same 32 rows, acc[db] the dims 32 * db .. + 31 (rows) of y's columns.
// AHEAD: each LDS read is issued before the product in front of it (the compiler, short of registers, puts it behind).
template <typename T, int D, bool AHEAD = false>
__device__ __forceinline__ void accum_xt(const char* tile, int row0, const f32x16& y, f32x16 (&acc)[D / 32], int lane) {
  constexpr int RB = Frag<T, D>::RB;
  const int hf = lane >> 5;
  if constexpr (sizeof(T) == 2) {
    const int fr = lane & 15, part = (lane >> 4) & 1;
    union X { s16x4 p[2]; bf16x8 h; };
    auto read = [&](int s, int db) {
      const int row = row0 + 16 * s + 4 * hf + (fr >> 2);
      const int sw0 = swz<RB>(row), sw1 = swz<RB>(row + 8);
      const int ch = db * 4 + part * 2 + ((fr >> 1) & 1), sub = (fr & 1) * 8;
      X a;
      a.p[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_t*)(tile + row * RB + ((ch ^ sw0) << 4) + sub));
      a.p[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_t*)(tile + (row + 8) * RB + ((ch ^ sw1) << 4) + sub));
      return a;
    };
    if constexpr (AHEAD) {
      const Chunk yb[2] = {pack8(y, 0), pack8(y, 1)};
      X a = read(0, 0);
#pragma unroll
      for (int i = 0; i < 2 * (D / 32); ++i) {
        const int db = i % (D / 32);
        const X n = i + 1 < 2 * (D / 32) ? read((i + 1) / (D / 32), (i + 1) % (D / 32)) : a;
        __builtin_amdgcn_sched_barrier(0);
        acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.h, yb[i / (D / 32)].h, acc[db], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
        a = n;
      }
    } else {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const Chunk yb = pack8(y, s);
#pragma unroll
        for (int db = 0; db < D / 32; ++db) acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(read(s, db).h, yb.h, acc[db], 0, 0, 0);
      }
    }
  } else {
    const int c = lane & 31;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int row = row0 + 8 * (i / 4) + 4 * hf + i % 4;
      const int sw = swz<RB>(row);
#pragma unroll
      for (int db = 0; db < D / 32; ++db) {
        const float a = *reinterpret_cast<const float*>(tile + row * RB + (((db * 8 + (c >> 2)) ^ sw) << 4) + (c & 3) * 4);
        acc[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, y[i], acc[db], 0, 0, 0);
      }
    }
  }
}

// Store a C tile (column c is an output row, registers its dims) times mul at p, the lane's output row.  Lanes c and
// c + 32 hold alternate groups of 4 dims; bf16 rows trade groups, so that a lane writes 16 bytes at once.  Every lane
// of the wave comes here; `live` says whether its row is written.
template <typename T, int D>
__device__ __forceinline__ void store_cols(T* p, const f32x16 (&x)[D / 32], float mul, int Dlive, int hf, bool live) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int g = 0; g < 4; g += 2) {
        union { bf16 h[4]; unsigned u[2]; } lo, hi;   // dims 8 * g + 4 * hf .. and 8 * (g + 1) + 4 * hf ..
#pragma unroll
        for (int e = 0; e < 4; ++e) lo.h[e] = (bf16)(x[db][4 * g + e] * mul), hi.h[e] = (bf16)(x[db][4 * g + 4 + e] * mul);
        swap_halves(lo.u[0], hi.u[0]);
        swap_halves(lo.u[1], hi.u[1]);
        const int d = db * 32 + 8 * (g + hf);
        if (live && d < Dlive) *reinterpret_cast<uint4*>(p + d) = make_uint4(lo.u[0], lo.u[1], hi.u[0], hi.u[1]);
      }
  } else {
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = db * 32 + 8 * g + 4 * hf;
        if (live && d < Dlive)
          *reinterpret_cast<float4*>(p + d) = make_float4(x[db][4 * g] * mul, x[db][4 * g + 1] * mul, x[db][4 * g + 2] * mul,
                                                          x[db][4 * g + 3] * mul);
      }
  }
}

// Key pieces of a sequence in the split forward: whole 64-key tiles, at least `chunk` keys, at most `most` pieces.
__device__ __forceinline__ int piece_keys(int lk, int chunk, int most) {
  return max(chunk, ((lk + most - 1) / most + 63) & ~63);
}

// Work item t of the split forward = (sequence, row tile, key piece), sequences in order, a sequence's pieces of
// one row tile next to each other.  Returns false past the last item.  The whole wave searches, 64 sequences at a time.
struct Piece {
  Seq s;
  int piece;
};
__device__ __forceinline__ bool find_piece(const PackedArgs& a, int BM, int t, int lane, Piece& p) {
  int base = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int b = b0 + lane;
    int n = 0, pieces = 1, q0 = 0, k0 = 0, len = 0, lk = 0;
    if (b < a.B) {
      q0 = cu_at(a.cu_q, b, a.Mq), k0 = cu_at(a.cu_k, b, a.Mk);
      len = max(cu_at(a.cu_q, b + 1, a.Mq) - q0, 0);
      lk = max(cu_at(a.cu_k, b + 1, a.Mk) - k0, 0);
      const int lq = b == a.B - 1 ? a.Mq - q0 : len;   // the last one's rows and those behind
      const int keys = piece_keys(lk, a.chunk, a.nsplit);
      pieces = max(1, (lk + keys - 1) / keys);
      n = (int)(((long)lq * a.G + BM - 1) / BM) * pieces;
    }
    int sum = n;   // inclusive sum over the lanes
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(sum, o, 64);
      if (lane >= o) sum += v;
    }
    const unsigned long long over = __ballot(base + sum > t);
    if (over) {
      const int w = __builtin_ctzll(over);
      const int item = t - (base + __shfl(sum - n, w, 64)), pw = __shfl(pieces, w, 64);
      p.s.b = __builtin_amdgcn_readfirstlane(b0 + w);
      p.s.tile = __builtin_amdgcn_readfirstlane(item / pw);
      p.s.start = __builtin_amdgcn_readlane(q0, w), p.s.len = __builtin_amdgcn_readlane(len, w);
      p.s.start2 = __builtin_amdgcn_readlane(k0, w), p.s.len2 = __builtin_amdgcn_readlane(lk, w);
      p.piece = __builtin_amdgcn_readfirstlane(item % pw);
      return true;
    }
    base += __shfl(sum, 63, 64);
  }
  return false;
}

}  // namespace ogv
