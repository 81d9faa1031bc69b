// Dense attention of a training step, forward and backward.
//
// Sequence n has len tokens (packed: tokens cu[n] .. cu[n + 1] - 1 of [T, H, D]; batched: the first
// seq_lens[n] of [B, H, S, D]). Token i sees key j of its own sequence if j <= i or j < prefix[n]
// (causal), or every key. With s = scale q_i . k_j, then cap tanh(s / cap), then - slope_h |i - j|:
//   o_i = sum_j P_ij v_j,  P_ij = exp(s_ij - lse_i),  lse_i = log sum_j exp(s_ij).
// Backward, with dP_ij = do_i . v_j and D_i = do_i . o_i - dlse_i:
//   dv_j = sum_i P_ij do_i,  dS_ij = P_ij (dP_ij - D_i) (1 - tanh^2),
//   dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i.
// Two kernels: one owns queries (dq, and D_i on the way), one owns keys (dk, dv of a KV head over the
// query heads of its group). Each forms S and dP for itself, seven products instead of five, and no
// sum depends on the order in which workgroups run.
//
// All three use v_mfma_f32_32x32x16 with the owned rows as columns of the result: a lane owns one row,
// the accumulator of S^T (or S) is the B operand of the product that follows, and the tiles that the
// workgroup walks over lie in LDS, brought by DMA a tile ahead, read in rows and (transposed) in
// columns. A workgroup owns 128 rows, four waves 32 each; tiles have 64 rows. P and dS are rounded to
// the input type for their products (as the MFMA takes them; dS of few rows in two parts, kDenseFew): results are
// off by up to half a step of their weighted magnitudes more than with P and dS in 32 bits. Maxima, sums and
// accumulators are fp32.
//
// Tokens that a row does not see do not reach it: where only some rows of a tile see a key, infinities
// and NaN of what the zero weights would multiply are left out of the product and added to the rows
// that see them after the last tile.
//
// Bound by the products and the vector work of a wave following each other: two waves a SIMD (all that the
// registers allow) overlap them in part. 8192 tokens, 32 / 8 heads of 128, bf16, capped: forward 693 us (0.79
// PFLOP/s, MFMA busy 37% of the cycles, the vector unit 66%: a capped score takes two exponentials and a
// reciprocal), dq 852 us (three products, 0.97, 47 and 63%), dk and dv 1177 us (four, 0.93, 43 and 51%), their join
// 59 us (5.0 TB/s). Ten documents of up to 3500 tokens, 28 / 4 heads: 765 (41 and 43%), 974 (48 and 35%), 1468 (42
// and 31%) and 42 us. 4 x 77 tokens: 11, 13, 15 and 4 us, a chain of loads, products and stores. (Medians of 23
// launches in a row; the clock moves them: the forward's first three took 843 us, its last ten 668.)
// At heads of 128 the kernel of dk and dv keeps 11 registers in scratch memory with a cap and a bias, one with a cap
// alone; no other kernel does.
// Measured and not kept: the scores of the next tile beside the exponentials of this one (spilled: forward 2000 to
// 3000 us instead of 700 to 800; with 512 registers and one wave a SIMD 1290 to 1420), the products of half a tile
// instruction by instruction beside the exponentials of the other half (no spills; forward 815 us instead of 800 and
// 775 instead of 757, steadily at work, where the clock falls with the power drawn), two blocks of rows a wave
// with 512 registers (copies between register files and spills), a higher wave priority during the products (1%).
#include <type_traits>

#include "scores.h"

#include "../../include/tasft_amd.h"

namespace tasft {

#define TASFT_INLINE __attribute__((always_inline))

constexpr int kDenseRows = 128;  // rows that a workgroup owns
constexpr int kDenseTile = 64;   // rows of a tile that it walks over
template <int D>
constexpr int dense_step() { return D == 128 ? 32 : 64; }  // the same of the kernel of dk and dv
constexpr int kDenseRun = 4;     // groups that an XCD takes at a time, see dense_place
// dS in two parts, what its rounding left over in a product of its own, where few roundings make a result: for
// sequences of at most kDenseFew tokens (dq and dk of 2 to 11 tokens were off by 1.5 to 1.64 times what rounding the
// result alone is, elsewhere by 1.47), and as long as a call's rows of all heads and their keys make at most
// kDenseFewScores: that costs 10 us or so where the host bounds the call (4 x 77 tokens of 8 / 2 heads: dq 11.8 and
// 13.0 us, dk and dv 13.1 and 14.8, 2 x 512 of 32 / 8 24.6 and 31.1, 33 and 41, the calls 150 us with either; 64 x
// 256, which do without, would take 517 us instead of 466).
constexpr int kDenseFew = 32;
constexpr int64_t kDenseFewScores = 1 << 24;
constexpr float kDenseMove = 8.f;  // a new maximum moves the exp2 reference only if this far above it
constexpr float kDenseLn2 = 0.69314718055994531f;

// A [batch, token, head] view of contiguous rows: element strides.
struct DenseRows {
  uint16_t* p;
  int64_t s[3];
};

struct DenseParams {
  DenseRows q, k, v, o, go, gq, gk, gv;
  float* lse;         // strides (batch, token, head)
  int64_t sl[3];
  const float* glse;  // or null
  int64_t sgl[3];
  int8_t* rest;       // [row][Hq][D]: what out's rounding left over (dense_rest_of), or null
  float* less;        // [head][row]: what the exponentials' arguments are less than x mul
  float* di;          // and D
  float* part_k;      // [SG][row][Hkv][D], or null
  float* part_v;
  const int32_t* cu;        // packed, or null
  const int32_t* seq_lens;  // batched, or null
  const int32_t* prefix;    // or null
  ScoreParams sc;
  float scale;
  int64_t rows;  // rows of a head in all: T, or B S
  int N, T, Hq, Hkv, G, L;  // T: tokens packed, or of a batch entry
  int tiles;                // workgroups along a sequence
  int SG;                   // workgroups that share a KV head's query heads
  int causal;
  int few;                  // sequences of at most so many tokens take dS in two parts
};

struct DenseSeq {
  int b;      // batch entry
  int t0, t1; // its tokens, the last ones without a sequence's part
  int len, pre;
};

__device__ __forceinline__ DenseSeq dense_seq(const DenseParams& p, int n) {
  DenseSeq s;
  if (p.cu) {
    s.b = 0;
    s.t0 = min(max(p.cu[n], 0), p.T);
    s.t1 = min(max(p.cu[n + 1], s.t0), p.T);
    s.len = min(s.t1 - s.t0, p.L);
  } else {
    s.b = n;
    s.t0 = 0;
    s.t1 = p.T;
    s.len = p.seq_lens ? min(max(p.seq_lens[n], 0), p.T) : p.T;
  }
  s.pre = p.causal && p.prefix ? min(max(p.prefix[n], 0), s.len) : 0;
  return s;
}

template <class R>
__device__ __forceinline__ uint16_t* dense_at(R& r, const DenseSeq& s, int i, int h) {
  return r.p + s.b * r.s[0] + (int64_t)(s.t0 + i) * r.s[1] + h * r.s[2];
}

// The group and tile of a workgroup of dk and dv. A group's workgroups walk over the same queries and share an
// XCD's L2 (workgroup i runs on XCD i % 8). Groups are as narrow as that allows (the heads that a workgroup
// takes), so that every XCD gets some of every sequence, turned by one in each eight: else an XCD would get all
// first or all last heads. An XCD takes kDenseRun of its groups at a time, tile by tile: the longest columns of all
// of them first (in another order for each tile: workgroups go round an XCD's shader engines, and one would get
// the same group every time; ten documents, 28 / 4 heads: 2030 us without that, 1470 with; one group at a time
// 1500, and one sequence of 8192 5% slower).
struct DensePlace {
  int group, tile;
};
__device__ __forceinline__ DensePlace dense_place(int64_t groups, int tiles) {
  const int64_t idx = blockIdx.x;
  const bool xcds = (groups & 7) == 0;
  const int64_t j = xcds ? idx >> 3 : idx, each = xcds ? groups >> 3 : groups;  // of an XCD
  const int64_t run = j / (kDenseRun * tiles), r = j - run * (kDenseRun * tiles);
  const int here = (int)min((int64_t)kDenseRun, each - run * kDenseRun);
  const int tile = (int)(r / here);
  const int64_t g = run * kDenseRun + (r + tile) % here;
  return {(int)(xcds ? 8 * g + ((idx + g) & 7) : g), tile};
}

// The kernel's argument read again: what only the end of a kernel uses is not kept in scalar registers over
// its main loop (they spilled).
typedef const __attribute__((address_space(4))) DenseParams* DenseParamsPtr;
__device__ __forceinline__ DenseParamsPtr dense_params_again() {
  DenseParamsPtr p = (DenseParamsPtr)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

// Rows of a head that no sequence has: those behind its length in tile `tile` of the workgroup's
// sequence, those that max_seqlen cuts off, and those behind the last sequence, shared out.
template <class F>
__device__ __forceinline__ void dense_rest(const DenseParams& p, const DenseSeq& s, int n, int tile, int tid, F&& clear) {
  if (!p.cu) {
    const int from = max(tile * kDenseRows, s.len), to = min((tile + 1) * kDenseRows, p.T);
    for (int t = from; t < to; ++t) clear(s.b, t);
    return;
  }
  if (tile == 0)
    for (int t = s.t0 + s.len; t < s.t1; ++t) clear(0, t);
  const int64_t end = min(max(p.cu[p.N], 0), p.T);
  for (int64_t t = end + (int64_t)n * p.tiles + tile; t < p.T; t += (int64_t)p.N * p.tiles) clear(0, (int)t);
}

// A row of D values of a head set to 0 by D / 8 lanes.
template <int D>
__device__ __forceinline__ void dense_clear(const DenseRows& r, int b, int t, int h, int tid) {
  if (tid < D / 8) *(u32x4_t*)(r.p + b * r.s[0] + (int64_t)t * r.s[1] + h * r.s[2] + tid * 8) = (u32x4_t){0u, 0u, 0u, 0u};
}

// What a rounding to 16 bits leaves over, as the difference of the two values' fp32 words in a byte: in 256ths of
// the rounded value's last place. D_i = do_i . o_i goes into every dS of a row with one sign: with o as it was
// rounded, rows that see few keys had half again the error of all the other roundings together.
template <int DT>
constexpr int dense_rest_bits() { return DT == kF16 ? 5 : 8; }  // of a word, below the byte
template <int DT>
__device__ __forceinline__ uint32_t dense_rest_of(float x, uint32_t bits16) {
  constexpr int S = dense_rest_bits<DT>();
  const int left = (int)(__float_as_uint(x) - __float_as_uint(bits16_to_f32<DT>(bits16)));
  const int q = (left + (1 << (S - 1))) >> S;
  return (uint32_t)max(min(q, 127), -128) & 255u;
}
// (Infinities and NaN stay what they are, also where they came to a result after its rest.)
template <int DT>
__device__ __forceinline__ float dense_with_rest(uint32_t bits16, int q) {
  const uint32_t word = __float_as_uint(bits16_to_f32<DT>(bits16));
  return __uint_as_float((word & 0x7f800000u) == 0x7f800000u ? word : word + (uint32_t)(q * (1 << dense_rest_bits<DT>())));
}

// Position of 16-byte chunk cc of row r in LDS: of 16 consecutive rows the same chunk, and of 4
// consecutive rows (from a multiple of 4) any 64 bytes, lie in different banks.
template <int D>
__device__ __forceinline__ int dense_swz(int r, int cc) {
  return cc ^ (D == 128 ? ((r & 3) << 2 | ((r >> 2) & 3)) : (((r >> 1) & 1) << 2 | ((r >> 2) & 3)));
}

__device__ __forceinline__ void dense_barrier() { asm volatile("s_barrier" ::: "memory"); }

// A pair of 16-bit values with infinities and NaN replaced by 0.
template <int DT>
__device__ __forceinline__ uint32_t dense_finite2(uint32_t w) {
  constexpr uint32_t E = DT == kF16 ? 0x7c00u : 0x7f80u;
  if ((w & E) == E) w &= 0xffff0000u;
  if ((w & (E << 16)) == (E << 16)) w &= 0xffffu;
  return w;
}

// a + both of a pair of 16-bit values, in fp32.
template <int DT>
__device__ __forceinline__ float dense_add2(uint32_t w, float a) {
  if constexpr (DT == kF16) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), __builtin_bit_cast(f16x2, 0x3c003c00u), a, false);
  } else {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), __builtin_bit_cast(bf16x2, 0x3f803f80u), a, false);
  }
}

typedef uint16_t dense_u16x2_t __attribute__((ext_vector_type(2)));

// What one of four waves does with tiles of ROWS rows in LDS.
template <int D, int DT, int ROWS>
struct DenseTiles {
  static constexpr int KSTEPS = D / 16;
  static constexpr int DTILES = D / 32;
  static constexpr int ROWB = D * 2;
  static constexpr int TILE = ROWS * ROWB;
  static constexpr int RPU = 1024 / ROWB;            // rows of a 1 KB DMA unit
  static constexpr int UPW = ROWS / 4 / RPU;  // units of a wave's share of the copying
  static constexpr int CPR = ROWB / 16;

  // What a lane brings of a tile: its part of row `row` (of the first of the wave's units), in chunk `chunk`.
  struct Share {
    int row;    // in bytes, from the tile's first row
    int chunk;
    __device__ __forceinline__ Share(int64_t stride, int wave, int lane) {
      const int r = wave * UPW * RPU + lane / CPR;
      row = r * (int)stride * 2;
      chunk = dense_swz<D>(r, lane % CPR);
    }
  };
  // Rows `first` .. of a head's tensor into a tile; rows from `len` on arrive as zeros.
  static __device__ __forceinline__ void dma(uint8_t* tile, const uint16_t* base, int64_t stride, Share at, int first,
                                             int len, int wave) {
    const int rows = min(len - first, ROWS);
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        (void*)(base + (int64_t)first * stride), (short)0, rows > 0 ? (rows - 1) * (int)stride * 2 + ROWB : 0, 0x00020000);
    asm volatile("" : "+v"(at.chunk));  // formed again for every tile: the units' offsets are not kept
#pragma unroll
    for (int u = 0; u < UPW; ++u) {  // RPU rows on the swizzle changes by an exclusive or
      const int off = at.row + u * RPU * (int)stride * 2 + ((at.chunk ^ ((D == 128 ? u : 2 * u) & 3)) << 4);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (TASFT_LDS void*)(tile + (wave * UPW + u) * 1024), 16, off, 0, 0, 0);
    }
  }
  // Where a lane reads in a tile. The swizzle moves 16-byte chunks by exclusive or within a row and repeats
  // every 16 rows, so that every other place is this one with constants: xor within the row, plus whole rows.
  struct Place {
    int rows;     // row lane % 32, chunk lane / 32
    int columns;  // row 4 (lane / 32) + (lane % 16) / 4, dims 16 (lane / 16 % 2) + 4 (lane % 4) .. + 3
    __device__ __forceinline__ Place(int lane) {
      const int col = lane & 31, half = lane >> 5, row = 4 * half + ((lane & 15) >> 2);
      rows = col * ROWB + dense_swz<D>(col, half) * 16;
      columns = row * ROWB + dense_swz<D>(row, 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) * 16 + (lane & 1) * 8;
    }
  };
  // Rows r0 .. r0 + 31 as the A operand, times b: 32 x 32 products. PARTS > 1: for kernels short of registers;
  // the operand is read in as many pieces, and its places are formed again for each use.
  template <int PARTS = 1>
  static __device__ __forceinline__ f32x16_t rows_times(const uint8_t* tile, int r0, const u32x4_t (&b)[KSTEPS], Place at) {
    constexpr int N = KSTEPS / PARTS;
    if (PARTS > 1) asm volatile("" : "+v"(at.rows));
    f32x16_t s = (f32x16_t){};
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
      u32x4_t a[N];
#pragma unroll
      for (int k = 0; k < N; ++k)
        a[k] = *(const u32x4_t*)(tile + (at.rows ^ (part * N + k) << 5) + r0 * ROWB);
#pragma unroll
      for (int k = 0; k < N; ++k) s = mfma16<DT>(a[k], b[part * N + k], s);
      if (PARTS > 1) __builtin_amdgcn_sched_barrier(0);
    }
    return s;
  }
  // Rows r0 .. r0 + 31 as the A operand, times rows c0 .. c0 + 31 of another tile as the B operand.
  static __device__ __forceinline__ f32x16_t rows_times_rows(const uint8_t* tile, int r0, const uint8_t* other, int c0,
                                                             Place at) {
    f32x16_t s = (f32x16_t){};
#pragma unroll
    for (int k = 0; k < KSTEPS; ++k) {
      const u32x4_t a = *(const u32x4_t*)(tile + (at.rows ^ k << 5) + r0 * ROWB);
      const u32x4_t b = *(const u32x4_t*)(other + (at.rows ^ k << 5) + c0 * ROWB);
      s = mfma16<DT>(a, b, s);
    }
    return s;
  }
  // acc [D x 32] += (rows r0 .. r0 + 31)^T b, b in the order of an accumulator's registers. With
  // `mixed` infinities and NaN are left out, and noted in `found` (in LDS: as a value it had the compiler
  // make a second copy of the loop for it, and spill).
  template <int PARTS = 1>
  static __device__ __forceinline__ void columns_times(const uint8_t* tile, int r0, const u32x4_t (&b)[2], bool mixed,
                                                       f32x16_t (&acc)[DTILES], Place at, int* found) {
    constexpr int N = 2 / PARTS;
    if (PARTS > 1) asm volatile("" : "+v"(at.columns));
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
      u32x2_t lo[N][DTILES], hi[N][DTILES];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const uint8_t* from = tile + (r0 + 16 * (part * N + e)) * ROWB;
#pragma unroll
        for (int dt = 0; dt < DTILES; ++dt) {  // 8 rows on the swizzle's bit 1 changes too
          lo[e][dt] = ds_read_tr16_b64((const void*)(from + (at.columns ^ dt << 6)));
          hi[e][dt] = ds_read_tr16_b64((const void*)(from + (at.columns ^ (dt << 6 | 32)) + 8 * ROWB));
        }
      }
      if (mixed) {
        asm volatile("");
        dense_u16x2_t top = {0, 0};  // the largest magnitudes tell whether there is one
#pragma unroll
        for (int e = 0; e < N; ++e)
#pragma unroll
          for (int dt = 0; dt < DTILES; ++dt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              top = __builtin_elementwise_max(top, __builtin_bit_cast(dense_u16x2_t, lo[e][dt][j] & 0x7fff7fffu));
              top = __builtin_elementwise_max(top, __builtin_bit_cast(dense_u16x2_t, hi[e][dt][j] & 0x7fff7fffu));
            }
        constexpr uint16_t E = DT == kF16 ? 0x7c00 : 0x7f80;
        if (__ballot(top[0] >= E || top[1] >= E)) {
          *found = 1;
#pragma unroll
          for (int e = 0; e < N; ++e)
#pragma unroll
            for (int dt = 0; dt < DTILES; ++dt)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                lo[e][dt][j] = dense_finite2<DT>(lo[e][dt][j]);
                hi[e][dt][j] = dense_finite2<DT>(hi[e][dt][j]);
              }
        }
      }
#pragma unroll
      for (int e = 0; e < N; ++e)
#pragma unroll
        for (int dt = 0; dt < DTILES; ++dt) {
          const u32x4_t a = {lo[e][dt][0], lo[e][dt][1], hi[e][dt][0], hi[e][dt][1]};
          acc[dt] = mfma16<DT>(a, b[part * N + e], acc[dt]);
        }
      if (PARTS > 1) __builtin_amdgcn_sched_barrier(0);
    }
  }
  // a + the sum of packed values.
  static __device__ __forceinline__ float sum(const u32x4_t (&b)[2], float a) {
#pragma unroll
    for (int pp = 0; pp < 2; ++pp)
#pragma unroll
      for (int j = 0; j < 4; ++j) a = dense_add2<DT>(b[pp][j], a);
    return a;
  }
  // The registers of a 32 x 32 product as the B operand of columns_times.
  static __device__ __forceinline__ void pack(u32x4_t (&b)[2], const f32x16_t& s) {
#pragma unroll
    for (int pp = 0; pp < 2; ++pp)
      b[pp] = (u32x4_t){pack16x2<DT>(s[8 * pp], s[8 * pp + 1]), pack16x2<DT>(s[8 * pp + 2], s[8 * pp + 3]),
                        pack16x2<DT>(s[8 * pp + 4], s[8 * pp + 5]), pack16x2<DT>(s[8 * pp + 6], s[8 * pp + 7])};
  }
  // What packing left over, packed (nothing of infinities).
  static __device__ __forceinline__ void pack_rest(u32x4_t (&b)[2], const f32x16_t& s, const u32x4_t (&had)[2]) {
#pragma unroll
    for (int pp = 0; pp < 2; ++pp)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t w = had[pp][j];
        b[pp][j] = dense_finite2<DT>(pack16x2<DT>(s[8 * pp + 2 * j] - bits16_to_f32<DT>(w & 0xffffu),
                                                  s[8 * pp + 2 * j + 1] - bits16_to_f32<DT>(w >> 16)));
      }
  }
  // A wave's 32 rows of the transposed accumulators times f, to `out` (row `col` at element `at`, < 0:
  // not there), whole rows through 32 rows of LDS of its own.
  static __device__ __forceinline__ void store(uint8_t* lds, const f32x16_t (&acc)[DTILES], float f, uint16_t* out,
                                               int64_t at, int lane) {
    const int col = lane & 31, half = lane >> 5;
#pragma unroll
    for (int dt = 0; dt < DTILES; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d0 = dt * 32 + 8 * g + 4 * half;
        const u32x2_t w = {pack16x2<DT>(acc[dt][4 * g] * f, acc[dt][4 * g + 1] * f),
                           pack16x2<DT>(acc[dt][4 * g + 2] * f, acc[dt][4 * g + 3] * f)};
        *(u32x2_t*)(lds + col * ROWB + (((d0 >> 3) ^ (col & (CPR - 1))) << 4) + (d0 & 7) * 2) = w;
      }
#pragma unroll
    for (int j = 0; j < 32 * CPR / kWave; ++j) {
      const int r = j * (kWave / CPR) + lane / CPR, c = lane % CPR;
      const u32x4_t x = *(const u32x4_t*)(lds + r * ROWB + ((c ^ (r & (CPR - 1))) << 4));
      const int64_t to = __shfl(at, r, kWave);
      if (to >= 0) *(u32x4_t*)(out + to + c * 8) = x;
    }
  }
  // A row as the B operand: dims 16 ks + 8 half .. + 7.
  static __device__ __forceinline__ void load_row(u32x4_t (&f)[KSTEPS], const uint16_t* row, int half) {
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks) f[ks] = *(const u32x4_t*)(row + half * 8 + ks * 16);
  }
  // The product of a row in memory and one held as the B operand.
  static __device__ __forceinline__ float dot(const uint16_t* row, const u32x4_t (&f)[KSTEPS], int half) {
    float sum = 0.f;
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks) {
      float x[8], y[8];
      unpack16x8<DT>(*(const u32x4_t*)(row + half * 8 + ks * 16), x);
      unpack16x8<DT>(f[ks], y);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(x[j], y[j], sum);
    }
    return pair_sum32(sum);
  }
  // The same with what a rounding left over of the row in memory added to it.
  static __device__ __forceinline__ float dot(const uint16_t* row, const int8_t* rest, const u32x4_t (&f)[KSTEPS], int half) {
    float sum = 0.f;
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks) {
      const u32x4_t x = *(const u32x4_t*)(row + half * 8 + ks * 16);
      const u32x2_t q = *(const u32x2_t*)(rest + half * 8 + ks * 16);
      float y[8];
      unpack16x8<DT>(f[ks], y);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        sum = fmaf(dense_with_rest<DT>(x[j >> 1] >> (16 * (j & 1)) & 0xffffu, (int8_t)(q[j >> 2] >> (8 * (j & 3)))), y[j], sum);
    }
    return pair_sum32(sum);
  }
  static __device__ __forceinline__ bool has_nonfinite(const uint16_t* row, int lane) {
    const uint32_t w = *(const uint32_t*)(row + (lane * 2) % D);
    return __ballot(dense_finite2<DT>(w) != w) != 0;
  }
};

// What follows the last tile where infinities or NaN were left out of a product: they are added to the stored
// results, key by key, from memory, for the rows that see them. (The sum is infinite or NaN, whatever its
// finite part; where another tile had them in its product, once more changes nothing.) Rolled loops: in the
// registers of the main loop's sums this took hundreds of spills there.
template <int D, int DT>
__device__ __forceinline__ float dense_dot(const uint16_t* a, const uint16_t* b) {
  float sum = 0.f;
#pragma nounroll
  for (int c = 0; c < D; c += 2) {
    const uint32_t x = *(const uint32_t*)(a + c), y = *(const uint32_t*)(b + c);
    sum = fmaf(bits16_to_f32<DT>(x & 0xffffu), bits16_to_f32<DT>(y & 0xffffu), sum);
    sum = fmaf(bits16_to_f32<DT>(x >> 16), bits16_to_f32<DT>(y >> 16), sum);
  }
  return sum;
}
// out (16-bit, or fp32 sums) += w x where x is infinite or NaN.
template <int D, int DT, class T>
__device__ __forceinline__ void dense_patch(T* out, const uint16_t* x, float w, int half) {
#pragma nounroll
  for (int d = half * (D / 2); d < (half + 1) * (D / 2); ++d) {
    const uint32_t b = x[d];
    if (dense_finite2<DT>(b) == b) continue;
    if constexpr (sizeof(T) == 2) out[d] = f32_to16<DT>(bits16_to_f32<DT>(out[d]) + w * bits16_to_f32<DT>(b));
    else out[d] += w * bits16_to_f32<DT>(b);
  }
}

// For each of the products s of 32 rows f(register, x, g), into s: x rises with the score (scores.h), g is a
// quarter of the cap's derivative, 1 - tanh^2 = 4 (r - r^2) with r = -gate. Distance of register rr:
// |d + off(rr)|; slope in units of x.
template <bool CAP, bool BIAS, class F>
__device__ __forceinline__ void dense_weights(f32x16_t& s, const ScoreParams& sc, float slope, float d, F&& f) {
  auto each = [&](auto score) TASFT_INLINE {
#pragma unroll
    for (int rr = 0; rr < 16; ++rr) {
      float g = 1.f, x = s[rr];
      if constexpr (CAP) {
        const float gate = cap_gate(s[rr], sc);
        x = score(s[rr], gate);
        g = fmaf(-gate, gate, -gate);
      }
      if constexpr (BIAS) x = fmaf(-slope, fabsf(d + (float)(8 * (rr >> 2) + (rr & 3))), x);
      s[rr] = f(rr, x, g);
    }
  };
  if (CAP && (BIAS || sc.cap_score)) each([&](float a, float gate) { return cap_score(a, gate, sc); });
  else each([](float, float gate) { return gate; });
}

// One score as above.
template <bool CAP, bool BIAS>
__device__ __forceinline__ float dense_score(float s, float& g, const ScoreParams& sc, float slope, float d) {
  float x = s;
  g = 1.f;
  if constexpr (CAP) {
    const float gate = cap_gate(s, sc);
    x = sc.cap_score ? cap_score(s, gate, sc) : gate;
    g = fmaf(-gate, gate, -gate);
  }
  return BIAS ? fmaf(-slope, fabsf(d), x) : x;
}

// ------------------------------------------------------------------------------------ forward
template <int D, int DT, bool CAP, bool BIAS>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) dense_fwd_kernel(const DenseParams p) {
  using X = DenseTiles<D, DT, kDenseTile>;
  __shared__ __attribute__((aligned(1024))) uint8_t k0_lds[X::TILE];
  __shared__ __attribute__((aligned(1024))) uint8_t v0_lds[X::TILE];
  __shared__ __attribute__((aligned(1024))) uint8_t k1_lds[X::TILE];
  __shared__ __attribute__((aligned(1024))) uint8_t v1_lds[X::TILE];
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid & 63;
  if (tid == 0) found = 0;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const typename X::Place place(lane);
  // The query heads of a KV head share an XCD's L2.
  int64_t group;
  int member;
  xcd_group_map(blockIdx.x, (int64_t)p.N * p.Hkv, p.tiles * p.G, &group, &member);
  const int n = (int)(group / p.Hkv), kvh = (int)(group % p.Hkv), h = kvh * p.G + member % p.G;
  const int tile = p.tiles - 1 - member / p.G;  // the longest rows first
  const DenseSeq sq = dense_seq(p, n);
  dense_rest(p, sq, n, tile, tid, [&](int b, int t) {
    dense_clear<D>(p.o, b, t, h, tid);
    if (tid == 0 && p.lse) p.lse[b * p.sl[0] + t * p.sl[1] + h * p.sl[2]] = -INFINITY;
  });
  const int r0 = tile * kDenseRows;
  if (r0 >= sq.len) return;
  const int i_first = r0 + wave * 32, i_last = min(i_first + 31, sq.len - 1), i_end = min(r0 + kDenseRows, sq.len) - 1;
  const bool row_ok = i_first + col < sq.len;
  const int i = min(i_first + col, sq.len - 1);
  // Keys a row sees: 0 .. lim. All rows of the wave see the keys to all_see, none one past any_see.
  auto sees = [&](int row) { return p.causal ? max(row, sq.pre - 1) : sq.len - 1; };
  const int lim = sees(i), all_see = sees(min(i_first, i_last)), any_see = i_first <= i_last ? sees(i_last) : -1;
  const int tiles = sees(i_end) / kDenseTile + 1;

  u32x4_t qf[X::KSTEPS];
  X::load_row(qf, dense_at(p.q, sq, i, h), half);
  const float slope = BIAS ? p.sc.slopes[h] * p.sc.slope_mul : 0.f;
  const uint16_t* kbase = dense_at(p.k, sq, 0, kvh);
  const uint16_t* vbase = dense_at(p.v, sq, 0, kvh);
  const typename X::Share koff(p.k.s[1], wave, lane), voff(p.v.s[1], wave, lane);
  auto bring = [&](uint8_t* kt, uint8_t* vt, int t) TASFT_INLINE {
    X::dma(kt, kbase, p.k.s[1], koff, t * kDenseTile, sq.len, wave);
    X::dma(vt, vbase, p.v.s[1], voff, t * kDenseTile, sq.len, wave);
  };

  f32x16_t oacc[X::DTILES];
#pragma unroll
  for (int dt = 0; dt < X::DTILES; ++dt) oacc[dt] = (f32x16_t){};
  // The weights' sum, for the log-sum, and their sum as they were rounded, for the output: its error is then of
  // what is added up less its mean, none where one key has all the weight (and D's, with the output, too: out was off
  // by up to 1.24 times its own rounding without it and is by 1.17, dq by 1.50 and 1.47; 782 us became 801).
  float m_ref = -INFINITY, l_run = 0.f, l_out = 0.f;

  auto step = [&](const uint8_t* ka, const uint8_t* va, uint8_t* kb, uint8_t* vb, int t) TASFT_INLINE {
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    dense_barrier();
    if (t + 1 < tiles) bring(kb, vb, t + 1);
    const int key0 = t * kDenseTile;
    if (key0 > any_see) return;
    const bool mixed = key0 + kDenseTile - 1 > all_see;
    f32x16_t s0 = X::rows_times(ka, 0, qf, place), s1 = X::rows_times(ka, 32, qf, place);
    if constexpr (CAP || BIAS) {
      const float d = (float)(key0 + 4 * half - i);
      auto same = [](int, float x, float) { return x; };
      dense_weights<CAP, BIAS>(s0, p.sc, slope, d, same);
      dense_weights<CAP, BIAS>(s1, p.sc, slope, d + 32.f, same);
    }
    if (mixed) {
      asm volatile("");  // a branch, no selections in other tiles
      const int lim0 = lim - key0 - 4 * half, lim1 = lim0 - 32;
#pragma unroll
      for (int rr = 0; rr < 16; ++rr) {
        const int off = 8 * (rr >> 2) + (rr & 3);
        s0[rr] = off > lim0 ? -INFINITY : s0[rr];
        s1[rr] = off > lim1 ? -INFINITY : s1[rr];
      }
    }
    float ma = fmaxf(fmaxf(s0[0], s0[1]), s0[2]), mb = fmaxf(fmaxf(s1[0], s1[1]), s1[2]);
#pragma unroll
    for (int rr = 3; rr < 15; rr += 2) {
      ma = fmaxf(fmaxf(ma, s0[rr]), s0[rr + 1]);
      mb = fmaxf(fmaxf(mb, s1[rr]), s1[rr + 1]);
    }
    const float mloc = fmaf(pair_max32(fmaxf(fmaxf(ma, s0[15]), fmaxf(mb, s1[15]))), p.sc.mul, CAP ? p.sc.add : 0.f);
    const bool move = mloc > m_ref + kDenseMove;
    if (__ballot(move)) {
      const float alpha = move ? __builtin_amdgcn_exp2f(m_ref - mloc) : 1.f;
      l_run *= alpha;
      l_out *= alpha;
#pragma unroll
      for (int dt = 0; dt < X::DTILES; ++dt) oacc[dt] *= alpha;
      m_ref = move ? mloc : m_ref;
    }
    const float less = (m_ref == -INFINITY ? 0.f : m_ref) - (CAP ? p.sc.add : 0.f);
    float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
    for (int rr = 0; rr < 16; ++rr) {
      s0[rr] = __builtin_amdgcn_exp2f(fmaf(s0[rr], p.sc.mul, -less));
      s1[rr] = __builtin_amdgcn_exp2f(fmaf(s1[rr], p.sc.mul, -less));
      sum0 += s0[rr];
      sum1 += s1[rr];
    }
    l_run += sum0 + sum1;
#pragma unroll
    for (int t2 = 0; t2 < 2; ++t2) {
      u32x4_t pb[2];
      X::pack(pb, t2 ? s1 : s0);
      l_out = X::sum(pb, l_out);
      X::columns_times(va, 32 * t2, pb, mixed, oacc, place, &found);
    }
  };
  bring(k0_lds, v0_lds, 0);
  for (int t = 0; t < tiles; t += 2) {
    step(k0_lds, v0_lds, k1_lds, v1_lds, t);
    if (t + 1 >= tiles) break;
    step(k1_lds, v1_lds, k0_lds, v0_lds, t + 1);
  }

  const DenseParamsPtr pe = dense_params_again();
  const float l_tot = pair_sum32(l_run);
  if (pe->lse && row_ok && half == 0)
    pe->lse[sq.b * pe->sl[0] + (sq.t0 + i) * pe->sl[1] + h * pe->sl[2]] = (m_ref + __builtin_amdgcn_logf(l_tot)) * kDenseLn2;
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  dense_barrier();                     // every wave is done with the tiles
  uint8_t* ost = ((wave & 2) ? v0_lds : k0_lds) + (wave & 1) * (32 * X::ROWB);
  const float l_div = pair_sum32(l_out), inv = 1.f / (l_div > 0.f ? l_div : 1.f);
  X::store(ost, oacc, inv, dense_at(pe->o, sq, 0, h), row_ok ? (int64_t)i * pe->o.s[1] : -1, lane);
  if (pe->rest && row_ok) {
    int8_t* to = pe->rest + (((int64_t)sq.b * pe->T + sq.t0 + i) * pe->Hq + h) * D + 4 * half;
#pragma unroll
    for (int dt = 0; dt < X::DTILES; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        uint32_t q = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = oacc[dt][4 * g + e] * inv;
          q |= dense_rest_of<DT>(x, f32_to16<DT>(x)) << (8 * e);
        }
        *(uint32_t*)(to + dt * 32 + 8 * g) = q;
      }
  }

  if (found) {
    __threadfence();
    const float less = m_ref + __builtin_amdgcn_logf(l_tot) - pe->sc.add;
#pragma nounroll
    for (int key = (all_see + 1) / kDenseTile * kDenseTile; key <= any_see; ++key) {
      const uint16_t* vr = vbase + (int64_t)key * pe->v.s[1];
      if (!X::has_nonfinite(vr, lane) || !row_ok || key > lim) continue;
      float gate;
      const float s = dense_score<CAP, BIAS>(dense_dot<D, DT>(dense_at(pe->q, sq, i, h), kbase + (int64_t)key * pe->k.s[1]),
                                             gate, p.sc, slope, (float)(key - i));
      dense_patch<D, DT>(dense_at(pe->o, sq, i, h), vr, __builtin_amdgcn_exp2f(fmaf(s, pe->sc.mul, -less)), half);
    }
  }
}

// ------------------------------------------------------------------------- backward: queries
template <int D, int DT, bool CAP, bool BIAS>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) dense_dq_kernel(const DenseParams p) {
  using X = DenseTiles<D, DT, kDenseTile>;
  __shared__ __attribute__((aligned(1024))) uint8_t k0_lds[X::TILE];
  __shared__ __attribute__((aligned(1024))) uint8_t v0_lds[X::TILE];
  __shared__ __attribute__((aligned(1024))) uint8_t k1_lds[X::TILE];
  __shared__ __attribute__((aligned(1024))) uint8_t v1_lds[X::TILE];
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid & 63;
  if (tid == 0) found = 0;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const typename X::Place place(lane);
  // The query heads of a KV head share an XCD's L2.
  int64_t group;
  int member;
  xcd_group_map(blockIdx.x, (int64_t)p.N * p.Hkv, p.tiles * p.G, &group, &member);
  const int n = (int)(group / p.Hkv), kvh = (int)(group % p.Hkv), h = kvh * p.G + member % p.G;
  const int tile = p.tiles - 1 - member / p.G;
  const DenseSeq sq = dense_seq(p, n);
  dense_rest(p, sq, n, tile, tid, [&](int b, int t) { dense_clear<D>(p.gq, b, t, h, tid); });
  const int r0 = tile * kDenseRows;
  if (r0 >= sq.len) return;
  const int i_first = r0 + wave * 32, i_last = min(i_first + 31, sq.len - 1), i_end = min(r0 + kDenseRows, sq.len) - 1;
  const bool row_ok = i_first + col < sq.len;
  const int i = min(i_first + col, sq.len - 1);
  auto sees = [&](int row) { return p.causal ? max(row, sq.pre - 1) : sq.len - 1; };
  const int lim = sees(i), all_see = sees(min(i_first, i_last)), any_see = i_first <= i_last ? sees(i_last) : -1;
  const int tiles = sees(i_end) / kDenseTile + 1;

  const uint16_t* kbase = dense_at(p.k, sq, 0, kvh);
  const uint16_t* vbase = dense_at(p.v, sq, 0, kvh);
  const typename X::Share koff(p.k.s[1], wave, lane), voff(p.v.s[1], wave, lane);
  auto bring = [&](uint8_t* kt, uint8_t* vt, int t) TASFT_INLINE {
    X::dma(kt, kbase, p.k.s[1], koff, t * kDenseTile, sq.len, wave);
    X::dma(vt, vbase, p.v.s[1], voff, t * kDenseTile, sq.len, wave);
  };
  bring(k0_lds, v0_lds, 0);

  u32x4_t qf[X::KSTEPS], gf[X::KSTEPS];
  X::load_row(qf, dense_at(p.q, sq, i, h), half);
  X::load_row(gf, dense_at(p.go, sq, i, h), half);
  const int64_t li = sq.b * p.sl[0] + (sq.t0 + i) * p.sl[1] + h * p.sl[2];
  // What the exponential's argument is less than x mul: with a cap the weights come four times as large, for its
  // derivative.
  const float less = fmaf(p.lse[li], kLog2e, CAP ? -2.f - p.sc.add : 0.f);
  float D_i = p.rest ? X::dot(dense_at(p.o, sq, i, h), p.rest + (((int64_t)sq.b * p.T + sq.t0 + i) * p.Hq + h) * D, gf, half)
                     : X::dot(dense_at(p.o, sq, i, h), gf, half);
  if (p.glse) D_i -= p.glse[sq.b * p.sgl[0] + (sq.t0 + i) * p.sgl[1] + h * p.sgl[2]];
  if (row_ok && half == 0) {
    const int64_t row = h * p.rows + (int64_t)sq.b * p.T + sq.t0 + i;
    p.less[row] = less;
    p.di[row] = D_i;
  }
  const float slope = BIAS ? p.sc.slopes[h] * p.sc.slope_mul : 0.f;

  f32x16_t acc[X::DTILES];
#pragma unroll
  for (int dt = 0; dt < X::DTILES; ++dt) acc[dt] = (f32x16_t){};
  auto step = [&](const uint8_t* ka, const uint8_t* va, uint8_t* kb, uint8_t* vb, int t) TASFT_INLINE {
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    dense_barrier();
    if (t + 1 < tiles) bring(kb, vb, t + 1);
#pragma unroll
    for (int t2 = 0; t2 < 2; ++t2) {
      const int key0 = t * kDenseTile + 32 * t2;
      if (key0 > any_see) continue;
      const bool mixed = key0 + 31 > all_see;
      f32x16_t s = X::rows_times(ka, 32 * t2, qf, place), dp = X::rows_times(va, 32 * t2, gf, place);
      dense_weights<CAP, BIAS>(s, p.sc, slope, (float)(key0 + 4 * half - i), [&](int rr, float x, float g) {
        const float w = __builtin_amdgcn_exp2f(fmaf(x, p.sc.mul, -less)) * (dp[rr] - D_i);
        return CAP ? w * g : w;
      });
      if (mixed) {
        asm volatile("");  // a branch, no selections in other tiles
        const int lim0 = lim - key0 - 4 * half;
#pragma unroll
        for (int rr = 0; rr < 16; ++rr) s[rr] = 8 * (rr >> 2) + (rr & 3) > lim0 ? 0.f : s[rr];
      }
      u32x4_t sb[2];
      X::pack(sb, s);
      if (sq.len <= p.few) {
        u32x4_t lo[2];
        X::pack_rest(lo, s, sb);
        X::columns_times(ka, 32 * t2, lo, mixed, acc, place, &found);
      }
      X::columns_times(ka, 32 * t2, sb, mixed, acc, place, &found);
    }
  };
  for (int t = 0; t < tiles; t += 2) {
    step(k0_lds, v0_lds, k1_lds, v1_lds, t);
    if (t + 1 >= tiles) break;
    step(k1_lds, v1_lds, k0_lds, v0_lds, t + 1);
  }

  const DenseParamsPtr pe = dense_params_again();
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  dense_barrier();                     // every wave is done with the tiles
  uint8_t* ost = ((wave & 2) ? v0_lds : k0_lds) + (wave & 1) * (32 * X::ROWB);
  X::store(ost, acc, pe->scale, dense_at(pe->gq, sq, 0, h), row_ok ? (int64_t)i * pe->gq.s[1] : -1, lane);

  if (found) {
    __threadfence();
#pragma nounroll
    for (int key = (all_see + 1) / kDenseTile * kDenseTile; key <= any_see; ++key) {
      const uint16_t* kr = kbase + (int64_t)key * pe->k.s[1];
      if (!X::has_nonfinite(kr, lane) || !row_ok || key > lim) continue;
      float gate;
      const float s = dense_score<CAP, BIAS>(dense_dot<D, DT>(dense_at(pe->q, sq, i, h), kr), gate, p.sc, slope,
                                             (float)(key - i));
      float ds = __builtin_amdgcn_exp2f(fmaf(s, pe->sc.mul, -less)) *
                 (dense_dot<D, DT>(dense_at(pe->go, sq, i, h), vbase + (int64_t)key * pe->v.s[1]) - D_i);
      ds *= gate;
      dense_patch<D, DT>(dense_at(pe->gq, sq, i, h), kr, ds * pe->scale, half);
    }
  }
}

// ---------------------------------------------------------------------------- backward: keys
template <int D, int DT, bool CAP, bool BIAS>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) dense_dkv_kernel(const DenseParams p) {
  constexpr int STEP = dense_step<D>();
  constexpr bool V_LDS = D == 128;
  using X = DenseTiles<D, DT, STEP>;
  using V = DenseTiles<D, DT, kDenseRows>;
  __shared__ __attribute__((aligned(1024))) uint8_t q0_lds[X::TILE];
  __shared__ __attribute__((aligned(1024))) uint8_t g0_lds[X::TILE];
  __shared__ __attribute__((aligned(1024))) uint8_t q1_lds[X::TILE];
  __shared__ __attribute__((aligned(1024))) uint8_t g1_lds[X::TILE];
  __shared__ __attribute__((aligned(1024))) uint8_t v_lds[V_LDS ? V::TILE : 16];
  __shared__ __attribute__((aligned(1024))) float st0_lds[2][kWave], st1_lds[2][kWave];  // lse, D
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid & 63;
  if (tid == 0) found = 0;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const typename X::Place place(lane);
  // Causal: the first keys are seen by the most rows.
  const DensePlace at = dense_place((int64_t)p.N * p.Hkv * p.SG, p.tiles);
  const int sg = at.group % p.SG, kvh = at.group / p.SG % p.Hkv, n = at.group / p.SG / p.Hkv, tile = at.tile;
  const DenseSeq sq = dense_seq(p, n);
  if (sg == 0)
    dense_rest(p, sq, n, tile, tid, [&](int b, int t) {
      dense_clear<D>(p.gk, b, t, kvh, tid);
      dense_clear<D>(p.gv, b, t, kvh, tid);
    });
  const int r0 = tile * kDenseRows;
  if (r0 >= sq.len) return;
  const int j_first = r0 + wave * 32, j_last = min(j_first + 31, sq.len - 1);
  const bool row_ok = j_first + col < sq.len;
  const int j = min(j_first + col, sq.len - 1);
  // The first query that sees a key. All of the wave's keys are seen by the rows from all_from on, none
  // by one before any_from.
  auto seen_from = [&](int key) { return p.causal && key >= sq.pre ? key : 0; };
  const int from = seen_from(j), all_from = seen_from(j_last), any_from = j_first <= j_last ? seen_from(j_first) : 0x7fffffff;
  const int t_first = seen_from(r0) / STEP, t_last = (sq.len - 1) / STEP;
  const int g_first = kvh * p.G + sg * p.G / p.SG, heads = kvh * p.G + (sg + 1) * p.G / p.SG - g_first;

  const typename X::Share qoff(p.q.s[1], wave, lane), goff(p.go.s[1], wave, lane);
  const int64_t row0 = (int64_t)sq.b * p.T + sq.t0;
  auto bring = [&](uint8_t* qt, uint8_t* gt, float (*st)[kWave], int h, int t) TASFT_INLINE {
    X::dma(qt, dense_at(p.q, sq, 0, h), p.q.s[1], qoff, t * STEP, sq.len, wave);
    X::dma(gt, dense_at(p.go, sq, 0, h), p.go.s[1], goff, t * STEP, sq.len, wave);
    if (wave < 2) {  // a row a lane (at D = 128 half of them are used); past the sequence's end zeros
      const int rows = min(sq.len - t * STEP, kWave);
      const float* from = (wave == 0 ? p.less : p.di) + h * p.rows + row0 + t * STEP;
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)from, (short)0, rows * 4, 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (TASFT_LDS void*)st[wave], 4, lane * 4, 0, 0, 0);
    }
  };
  bring(q0_lds, g0_lds, st0_lds, g_first, t_last);

  // K as the B operand in registers; V too, or at D = 128, where there is no room for it beside the sums, in LDS.
  u32x4_t kf[X::KSTEPS], vf[X::KSTEPS];
  X::load_row(kf, dense_at(p.k, sq, j, kvh), half);
  if constexpr (V_LDS)
    V::dma(v_lds, dense_at(p.v, sq, 0, kvh), p.v.s[1], typename V::Share(p.v.s[1], wave, lane), r0, sq.len, wave);
  else
    X::load_row(vf, dense_at(p.v, sq, j, kvh), half);
  f32x16_t ka[X::DTILES], va[X::DTILES];
#pragma unroll
  for (int dt = 0; dt < X::DTILES; ++dt) ka[dt] = va[dt] = (f32x16_t){};
  auto step = [&](const uint8_t* qa, const uint8_t* ga, const float (*st)[kWave], uint8_t* qb, uint8_t* gb,
                  float (*stb)[kWave], int h, int t, int hn, int tn) TASFT_INLINE {
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    dense_barrier();
    if (hn >= 0) bring(qb, gb, stb, hn, tn);
    const float slope = BIAS ? p.sc.slopes[h] * p.sc.slope_mul : 0.f;
#pragma unroll
    for (int t2 = 0; t2 < STEP / 32; ++t2) {
      const int i0 = t * STEP + 32 * t2;
      if (i0 + 31 < any_from || (STEP > 32 && i0 >= sq.len)) continue;
      const bool mixed = i0 < all_from;
      // Rows behind the sequence's end came as zeros, and make weights of the bias alone (or NaN of an infinite key).
      const bool cut = mixed || i0 + 31 >= sq.len;
      const float* less = st[0] + 32 * t2 + 4 * half;
      const float* di = st[1] + 32 * t2 + 4 * half;
      // Elements of rows that do not see the key become 0.
      auto keep = [&](f32x16_t& x) TASFT_INLINE {
        int first = from - i0 - 4 * half;
        const uint32_t rows = sq.len - from;
        asm volatile("" : "+v"(first));  // formed here, and a branch: no selections in other tiles
#pragma unroll
        for (int rr = 0; rr < 16; ++rr) x[rr] = (uint32_t)(8 * (rr >> 2) + (rr & 3) - first) < rows ? x[rr] : 0.f;
      };
      f32x16_t s = X::rows_times(qa, 32 * t2, kf, place), w;
      u32x4_t b[2];
      dense_weights<CAP, BIAS>(s, p.sc, slope, (float)(i0 + 4 * half - j), [&](int rr, float x, float g) {
        w[rr] = __builtin_amdgcn_exp2f(fmaf(x, p.sc.mul, -less[8 * (rr >> 2) + (rr & 3)]));
        return CAP ? w[rr] * g : w[rr];
      });
      if (cut) keep(w);
      X::pack(b, w);
      X::template columns_times<D == 128 ? 2 : 1>(ga, 32 * t2, b, mixed, va, place, &found);
      f32x16_t dp;
      if constexpr (V_LDS) dp = X::rows_times_rows(ga, 32 * t2, v_lds, wave * 32, place);
      else dp = X::rows_times(ga, 32 * t2, vf, place);
#pragma unroll
      for (int rr = 0; rr < 16; ++rr) s[rr] *= dp[rr] - di[8 * (rr >> 2) + (rr & 3)];
      if (cut) keep(s);
      X::pack(b, s);
      if (sq.len <= p.few) {
        u32x4_t lo[2];
        X::pack_rest(lo, s, b);
        X::template columns_times<D == 128 ? 2 : 1>(qa, 32 * t2, lo, mixed, ka, place, &found);
      }
      X::template columns_times<D == 128 ? 2 : 1>(qa, 32 * t2, b, mixed, ka, place, &found);
    }
  };
  // From the last rows, which every key's workgroup walks over, to the first: the workgroups of a group read the
  // same tiles at the same time.
  int h = g_first, t = t_last;
  const int steps = heads * (t_last - t_first + 1);
  for (int done = 0; done < steps; done += 2) {
    int hn = h, tn = t - 1;
    if (tn < t_first) tn = t_last, ++hn;
    step(q0_lds, g0_lds, st0_lds, q1_lds, g1_lds, st1_lds, h, t, done + 1 < steps ? hn : -1, tn);
    if (done + 1 >= steps) break;
    h = hn, t = tn - 1;
    if (t < t_first) t = t_last, ++h;
    step(q1_lds, g1_lds, st1_lds, q0_lds, g0_lds, st0_lds, hn, tn, done + 2 < steps ? h : -1, t);
  }

  const DenseParamsPtr pe = dense_params_again();
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  dense_barrier();                     // every wave is done with the tiles
  if (pe->SG > 1) {  // sums of these heads, joined by dense_join_kernel
    if (row_ok) {
      const int64_t at = (((int64_t)sg * pe->rows + row0 + j) * pe->Hkv + kvh) * D + 4 * half;
#pragma unroll
      for (int dt = 0; dt < X::DTILES; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int d0 = dt * 32 + 8 * g;
          const f32x16_t &x = ka[dt], &y = va[dt];
          *(f32x4_t*)(pe->part_k + at + d0) = (f32x4_t){x[4 * g], x[4 * g + 1], x[4 * g + 2], x[4 * g + 3]};
          *(f32x4_t*)(pe->part_v + at + d0) = (f32x4_t){y[4 * g], y[4 * g + 1], y[4 * g + 2], y[4 * g + 3]};
        }
    }
  } else {
    uint8_t* vst = (wave & 2 ? wave & 1 ? g1_lds : q1_lds : wave & 1 ? g0_lds : q0_lds);
    uint8_t* kst = V_LDS ? v_lds + wave * (32 * X::ROWB) : vst + 32 * X::ROWB;
    X::store(kst, ka, pe->scale, dense_at(pe->gk, sq, 0, kvh), row_ok ? (int64_t)j * pe->gk.s[1] : -1, lane);
    X::store(vst, va, CAP ? 0.25f : 1.f, dense_at(pe->gv, sq, 0, kvh), row_ok ? (int64_t)j * pe->gv.s[1] : -1, lane);
  }

  if (found) {
    __threadfence();
    // The rows before all_from, with those behind it in the last 32 of them.
    const int end = min((all_from + 31) / 32 * 32, sq.len);
#pragma nounroll
    for (int gh = g_first; gh < g_first + heads; ++gh) {
      const float slope = BIAS ? pe->sc.slopes[gh] * pe->sc.slope_mul : 0.f;
#pragma nounroll
      for (int i = any_from / 32 * 32; i < end; ++i) {
        const uint16_t* qr = dense_at(pe->q, sq, i, gh);
        const uint16_t* gr = dense_at(pe->go, sq, i, gh);
        const bool bad_q = X::has_nonfinite(qr, lane), bad_g = X::has_nonfinite(gr, lane);
        if (!bad_q && !bad_g) continue;
        const float less = pe->less[gh * pe->rows + row0 + i], di = pe->di[gh * pe->rows + row0 + i];
        if (!row_ok || i < from) continue;
        float gate;
        const float s = dense_score<CAP, BIAS>(dense_dot<D, DT>(qr, dense_at(pe->k, sq, j, kvh)), gate, p.sc, slope,
                                               (float)(i - j));
        const float w = __builtin_amdgcn_exp2f(fmaf(s, pe->sc.mul, -less));
        float ds = w * (dense_dot<D, DT>(gr, dense_at(pe->v, sq, j, kvh)) - di);
        ds *= gate;
        const int64_t at = (((int64_t)sg * pe->rows + row0 + j) * pe->Hkv + kvh) * D;
        if (bad_g) {
          if (pe->SG > 1) dense_patch<D, DT>(pe->part_v + at, gr, w, half);
          else dense_patch<D, DT>(dense_at(pe->gv, sq, j, kvh), gr, CAP ? 0.25f * w : w, half);
        }
        if (bad_q) {
          if (pe->SG > 1) dense_patch<D, DT>(pe->part_k + at, qr, ds, half);
          else dense_patch<D, DT>(dense_at(pe->gk, sq, j, kvh), qr, ds * pe->scale, half);
        }
      }
    }
  }
}

// Joins the SG partial sums of every key's gradients: D / 4 lanes a row.
template <int D, int DT, bool CAP>
__global__ void __launch_bounds__(256) dense_join_kernel(const DenseParams p) {
  constexpr int LPR = D / 4;
  const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LPR;
  const int c = threadIdx.x % LPR;
  const int64_t all = p.rows * p.Hkv;
  if (row >= all) return;
  const int64_t tok = row / p.Hkv;
  const int kvh = (int)(row - tok * p.Hkv);
  const int b = p.cu ? 0 : (int)(tok / p.T), t = p.cu ? (int)tok : (int)(tok - (int64_t)b * p.T);
  // Rows that no workgroup computed are zeros already; their partial sums are not written. (A packed row
  // that max_seqlen cuts off is found by its sequence.)
  if (!p.cu) {
    if (p.seq_lens && t >= p.seq_lens[b]) return;
  } else {
    int lo = 0, hi = p.N;  // the last sequence that starts at or before t
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      (p.cu[mid] <= t ? lo : hi) = mid;
    }
    const int t0 = max(p.cu[lo], 0);
    if (t >= min(p.cu[lo + 1], t0 + p.L) || t < t0) return;
  }
  const int64_t at = row * D + c * 4, step = all * D;
  f32x4_t k = *(const f32x4_t*)(p.part_k + at), v = *(const f32x4_t*)(p.part_v + at);
  for (int s = 1; s < p.SG; ++s) {
    k += *(const f32x4_t*)(p.part_k + at + s * step);
    v += *(const f32x4_t*)(p.part_v + at + s * step);
  }
  k *= p.scale;
  if (CAP) v *= 0.25f;  // (four times the weights, see dense_dq_kernel)
  *(u32x2_t*)(p.gk.p + b * p.gk.s[0] + (int64_t)t * p.gk.s[1] + kvh * p.gk.s[2] + c * 4) =
      (u32x2_t){pack16x2<DT>(k[0], k[1]), pack16x2<DT>(k[2], k[3])};
  *(u32x2_t*)(p.gv.p + b * p.gv.s[0] + (int64_t)t * p.gv.s[1] + kvh * p.gv.s[2] + c * 4) =
      (u32x2_t){pack16x2<DT>(v[0], v[1]), pack16x2<DT>(v[2], v[3])};
}

}  // namespace tasft

using namespace tasft;

static int dense_rows(DenseRows& r, const char* what, const char* name, const void* ptr, const int64_t* s) {
  if (!ptr || !s) return set_error(kErrInvalidArgument, "%s: null pointer argument", what);
  if (!strides_nonneg(s, 4)) return set_error(kErrInvalidArgument, "%s: strides of %s must be non-negative", what, name);
  if (s[3] != 1) return set_error(kErrInvalidArgument, "%s: head dims of %s must be contiguous", what, name);
  if ((s[0] & 7) || (s[1] & 7) || (s[2] & 7) || ((uintptr_t)ptr & 15))
    return set_error(kErrInvalidArgument, "%s: strides of %s must be multiples of 8 on a 16-byte aligned base", what, name);
  // (128 rows are addressed with 32-bit byte offsets.)
  if (s[2] >= (int64_t)1 << 23) return set_error(kErrUnsupported, "%s: token stride of %s too large", what, name);
  r.p = (uint16_t*)ptr;
  r.s[0] = s[0];
  r.s[1] = s[2];
  r.s[2] = s[1];
  return kOk;
}

// Workgroups that share a KV head's query heads, so that there are two rounds of the 512 that the GPU holds, and
// causal columns of unequal length even out: 4 x 2048 tokens of 32 / 8 heads backward and forward 819 us with one,
// 760 with two, 817 with four, 899 with three (two heads, one, one); 16 x 1024 (1024 workgroups already) 873 with
// one, 929 with two; ten ragged documents, 28 / 4 heads, 3930 and 3130. Their partial sums cost as much whatever
// the sequences' length, so that long ones take four rounds. In turn on one card, two rounds and four: ten documents
// 3150 us and 3620, 4 x 2048 capped and biased 957 and 1019, 2 x 4096 1256 and 1286, 8192 2357 and 2335 (capped 2757
// and 2723), 2 x 8192 4705 and 4641: little to gain beyond 6144, but to lose before it. Shares that would be of one
// and two heads become single heads.
static int dense_head_splits(int64_t rows, int64_t num_kv_heads, int64_t group, int64_t max_seqlen) {
  const int64_t wgs = (rows + kDenseRows - 1) / kDenseRows * num_kv_heads;
  const int64_t want = ((max_seqlen >= 6144 ? 2048 : 1024) + wgs - 1) / wgs;
  return (int)(2 * want > group && want > 1 ? group : want);
}

extern "C" size_t tasft_dense_bwd_workspace_bytes(int64_t num_seqs, int64_t rows, int64_t num_q_heads,
                                                  int64_t num_kv_heads, int64_t max_seqlen, int64_t head_dim) {
  if (num_seqs <= 0 || rows <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || max_seqlen <= 0 || head_dim <= 0 ||
      num_q_heads % num_kv_heads != 0)
    return 0;
  const int sg = dense_head_splits(rows, num_kv_heads, num_q_heads / num_kv_heads, max_seqlen);
  const size_t stats = ((size_t)rows * num_q_heads * 8 + 15) / 16 * 16;
  return stats + (sg > 1 ? (size_t)sg * rows * num_kv_heads * head_dim * 8 : 0);
}

static int dense_params(DenseParams& p, const char* what, const int32_t* cu, const int32_t* seq_lens,
                        const int32_t* prefix, const float* slopes, int64_t num_seqs, int64_t tokens,
                        int64_t num_q_heads, int64_t num_kv_heads, int64_t max_seqlen, int64_t head_dim, float scale,
                        float softcap, int causal, int dtype) {
  if (dtype != kBf16 && dtype != kF16)
    return set_error(kErrUnsupported, "%s: dtype must be bf16 (0) or fp16 (1), got %d", what, dtype);
  if (num_seqs <= 0 || tokens <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || max_seqlen <= 0)
    return set_error(kErrInvalidArgument, "%s: sizes must be positive", what);
  if (num_q_heads % num_kv_heads != 0)
    return set_error(kErrInvalidArgument, "%s: num_q_heads must be a multiple of num_kv_heads", what);
  if (head_dim != 64 && head_dim != 128)
    return set_error(kErrUnsupported, "%s: head_dim must be 64 or 128, got %lld", what, (long long)head_dim);
  if (!score_range(scale, softcap))
    return set_error(kErrInvalidArgument, "%s: scale must be positive, softcap not negative, and neither out of range", what);
  if (cu && seq_lens) return set_error(kErrInvalidArgument, "%s: cu_seqlens or seq_lens, not both", what);
  const int64_t lim = 0x7fffffff - 255;
  if (num_seqs > lim || tokens > lim || num_q_heads > 65535 || (!cu && num_seqs * tokens > ((int64_t)1 << 40)))
    return set_error(kErrUnsupported, "%s: sizes exceed 32 bits", what);
  p.cu = cu;
  p.seq_lens = seq_lens;
  p.prefix = prefix;
  p.sc = score_params(scale, softcap, slopes);
  p.scale = scale;
  p.rows = cu ? tokens : num_seqs * tokens;
  p.N = (int)num_seqs;
  p.T = (int)tokens;
  p.Hq = (int)num_q_heads;
  p.Hkv = (int)num_kv_heads;
  p.G = (int)(num_q_heads / num_kv_heads);
  p.L = (int)(max_seqlen < tokens && cu ? max_seqlen : tokens);
  p.tiles = (p.L + kDenseRows - 1) / kDenseRows;
  p.SG = 1;
  p.causal = causal;
  const int64_t few = kDenseFewScores / (p.rows * p.Hq);
  p.few = (int)(few < kDenseFew ? kDenseFew : few);
  // Launches of fewer than 2^32 threads.
  const int64_t most = 0xffffffffll / 256;
  if (num_seqs * num_q_heads > most || num_seqs * num_q_heads * p.tiles > most ||
      p.rows > most * 4 / num_kv_heads)
    return set_error(kErrUnsupported, "%s: launch too large", what);
  return kOk;
}

// Calls run(std::integral_constant D, DT, CAP, BIAS).
template <class F>
static void dense_dispatch(int64_t head_dim, int dtype, bool cap, bool bias, F&& run) {
  auto with_bias = [&](auto d, auto dt, auto c) {
    if (bias) run(d, dt, c, std::true_type{});
    else run(d, dt, c, std::false_type{});
  };
  auto with_cap = [&](auto d, auto dt) {
    if (cap) with_bias(d, dt, std::true_type{});
    else with_bias(d, dt, std::false_type{});
  };
  auto with_dtype = [&](auto d) {
    if (dtype == kF16) with_cap(d, std::integral_constant<int, kF16>{});
    else with_cap(d, std::integral_constant<int, kBf16>{});
  };
  if (head_dim == 128) with_dtype(std::integral_constant<int, 128>{});
  else with_dtype(std::integral_constant<int, 64>{});
}

extern "C" int tasft_dense_fwd(const void* q, const void* k, const void* v, void* out, float* lse, void* out_rest,
                               const int32_t* cu_seqlens, const int32_t* seq_lens, const int32_t* prefix_lens,
                               const float* alibi_slopes, int64_t num_seqs, int64_t tokens, int64_t num_q_heads,
                               int64_t num_kv_heads, int64_t max_seqlen, int64_t head_dim, const int64_t* q_strides,
                               const int64_t* k_strides, const int64_t* v_strides, const int64_t* o_strides,
                               const int64_t* lse_strides, float scale, float softcap, int causal, int dtype,
                               void* stream) {
  const char* what = "dense attention";
  DenseParams p = {};
  if (const int rc = dense_params(p, what, cu_seqlens, seq_lens, prefix_lens, alibi_slopes, num_seqs, tokens, num_q_heads,
                                  num_kv_heads, max_seqlen, head_dim, scale, softcap, causal, dtype))
    return rc;
  if (const int rc = dense_rows(p.q, what, "q", q, q_strides)) return rc;
  if (const int rc = dense_rows(p.k, what, "k", k, k_strides)) return rc;
  if (const int rc = dense_rows(p.v, what, "v", v, v_strides)) return rc;
  if (const int rc = dense_rows(p.o, what, "out", out, o_strides)) return rc;
  if (lse && (!lse_strides || !strides_nonneg(lse_strides, 3)))
    return set_error(kErrInvalidArgument, "dense attention: strides of lse must be non-negative");
  if ((uintptr_t)out_rest & 7) return set_error(kErrInvalidArgument, "dense attention: out_rest must be 8-byte aligned");
  p.rest = (int8_t*)out_rest;
  p.lse = lse;
  if (lse) p.sl[0] = lse_strides[0], p.sl[2] = lse_strides[1], p.sl[1] = lse_strides[2];
  const dim3 grid((unsigned)((int64_t)p.N * p.Hq * p.tiles));
  dense_dispatch(head_dim, dtype, softcap > 0.f, alibi_slopes != nullptr, [&](auto d, auto dt, auto c, auto b) {
    hipLaunchKernelGGL((dense_fwd_kernel<d.value, dt.value, c.value, b.value>), grid, dim3(256), 0, (hipStream_t)stream, p);
  });
  return check_launch(what);
}

extern "C" int tasft_dense_bwd(const void* q, const void* k, const void* v, const void* out, const float* lse,
                               const void* out_rest, const void* grad_out, const float* grad_lse, void* grad_q,
                               void* grad_k, void* grad_v, void* workspace, size_t workspace_bytes,
                               const int32_t* cu_seqlens, const int32_t* seq_lens, const int32_t* prefix_lens,
                               const float* alibi_slopes,
                               int64_t num_seqs, int64_t tokens, int64_t num_q_heads, int64_t num_kv_heads,
                               int64_t max_seqlen, int64_t head_dim, const int64_t* q_strides, const int64_t* k_strides,
                               const int64_t* v_strides, const int64_t* o_strides, const int64_t* lse_strides,
                               const int64_t* go_strides, const int64_t* glse_strides, const int64_t* gq_strides,
                               const int64_t* gk_strides, const int64_t* gv_strides, float scale, float softcap,
                               int causal, int dtype, void* stream) {
  const char* what = "dense attention backward";
  DenseParams p = {};
  if (const int rc = dense_params(p, what, cu_seqlens, seq_lens, prefix_lens, alibi_slopes, num_seqs, tokens, num_q_heads,
                                  num_kv_heads, max_seqlen, head_dim, scale, softcap, causal, dtype))
    return rc;
  if (const int rc = dense_rows(p.q, what, "q", q, q_strides)) return rc;
  if (const int rc = dense_rows(p.k, what, "k", k, k_strides)) return rc;
  if (const int rc = dense_rows(p.v, what, "v", v, v_strides)) return rc;
  if (const int rc = dense_rows(p.o, what, "out", out, o_strides)) return rc;
  if (const int rc = dense_rows(p.go, what, "grad_out", grad_out, go_strides)) return rc;
  if (const int rc = dense_rows(p.gq, what, "grad_q", grad_q, gq_strides)) return rc;
  if (const int rc = dense_rows(p.gk, what, "grad_k", grad_k, gk_strides)) return rc;
  if (const int rc = dense_rows(p.gv, what, "grad_v", grad_v, gv_strides)) return rc;
  if (!lse || !lse_strides || (grad_lse && !glse_strides))
    return set_error(kErrInvalidArgument, "dense attention backward: null pointer argument");
  if (!strides_nonneg(lse_strides, 3) || (grad_lse && !strides_nonneg(glse_strides, 3)))
    return set_error(kErrInvalidArgument, "dense attention backward: strides must be non-negative");
  if (!workspace || workspace_bytes < tasft_dense_bwd_workspace_bytes(num_seqs, p.rows, num_q_heads, num_kv_heads,
                                                                      max_seqlen, head_dim))
    return set_error(kErrWorkspace, "dense attention backward: workspace too small");
  if ((uintptr_t)workspace & 15)
    return set_error(kErrInvalidArgument, "dense attention backward: workspace must be 16-byte aligned");
  if ((uintptr_t)out_rest & 7)
    return set_error(kErrInvalidArgument, "dense attention backward: out_rest must be 8-byte aligned");
  p.rest = (int8_t*)out_rest;
  p.lse = (float*)lse;
  p.sl[0] = lse_strides[0], p.sl[2] = lse_strides[1], p.sl[1] = lse_strides[2];
  p.glse = grad_lse;
  if (grad_lse) p.sgl[0] = glse_strides[0], p.sgl[2] = glse_strides[1], p.sgl[1] = glse_strides[2];
  p.SG = dense_head_splits(p.rows, num_kv_heads, p.G, max_seqlen);  // as given: as the workspace's size was asked for
  p.less = (float*)workspace;
  p.di = p.less + p.rows * p.Hq;
  const size_t stats = ((size_t)p.rows * p.Hq * 8 + 15) / 16 * 16;
  if (p.SG > 1) {
    p.part_k = (float*)((uint8_t*)workspace + stats);
    p.part_v = p.part_k + (int64_t)p.SG * p.rows * p.Hkv * head_dim;
  }
  const dim3 grid_q((unsigned)((int64_t)p.N * p.Hq * p.tiles)), grid_k((unsigned)((int64_t)p.N * p.Hkv * p.tiles * p.SG));
  const hipStream_t st = (hipStream_t)stream;
  dense_dispatch(head_dim, dtype, softcap > 0.f, alibi_slopes != nullptr, [&](auto d, auto dt, auto c, auto b) {
    hipLaunchKernelGGL((dense_dq_kernel<d.value, dt.value, c.value, b.value>), grid_q, dim3(256), 0, st, p);
    hipLaunchKernelGGL((dense_dkv_kernel<d.value, dt.value, c.value, b.value>), grid_k,
                       dim3(256), 0, st, p);
    if (p.SG > 1) {
      const int64_t lanes = p.rows * p.Hkv * (d.value / 4);
      hipLaunchKernelGGL((dense_join_kernel<d.value, dt.value, c.value>), dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, st, p);
    }
  });
  return check_launch(what);
}
