// Attention of a chunk of new tokens over a paged cache.
//
// Sequence n of a packed batch has kv_len tokens in its pages, the last len of them new:
// token i of the chunk is at position p = kv_len - len + i and sees keys j <= p (causal), of
// key blocks its block mask selects if there is one:
//   o_i = softmax_j(q_i . k_j scale) v_j,   lse_i = log sum_j exp(q_i . k_j scale).
// A row that sees no key gives 0 and -inf.
//
// The rows of one KV head are its chunk's tokens times the query heads of its group: they share
// K and V. Dense: a workgroup takes a tile of 128 of them, in token order; four waves own 32 rows
// each and share 64-key tiles of K and V in LDS, brought by DMA through the page table a tile
// ahead: two stages, one barrier a tile. Masked: neighbouring heads and blocks see different keys,
// so a workgroup takes 64 positions of one head aligned to the mask's blocks, two waves, with one
// K and one V tile; but where all rows of a KV head fit one wave, the dense form goes over the tiles
// that any of them selects, each row with its own bits of the mask. S^T = K Q^T with
// v_mfma_f32_32x32x16, so a lane owns one row: its running maximum and sum stay in the lane (and the
// one 32 away), and the accumulator of S^T is the B operand of O^T = V^T P^T. P is rounded to the
// input type for that product (as the MFMA takes it): outputs are off by up to half a step of their
// weighted magnitudes more than with P in 32 bits. Maxima, sums, O and the log-sum are fp32.
//
// Masked scores are -inf before the exponential, and a key past kv_len is never read (its row
// arrives as zeros). A tile in which only some rows see a key could still carry an infinity or
// NaN of V into the others as 0 * inf: there V's largest magnitude is looked for (every value by
// itself took as long as the rest of the tile) and, if it is not finite, such values are left out of the
// product; after the last tile they are added key by key to the rows that see them. (A row that sees
// an infinity whose weight rounds to 0, in fp16 below 2^-25 of the row's largest, gets NaN.)
//
// Many rows: bound by the matrix cores and the exponentials of one wave not running beside the
// other's (two waves per SIMD, all the registers allow). 2048 tokens of 32 / 8 heads over 32768 keys:
// 1045 us, 1.02 PFLOP/s, 49% MFMA busy (1003 to 1082 by the card); a fifth of the blocks of 4 requests
// of 2048 over up to 16384: 360 us, 0.69 PFLOP/s, 34% busy (354 to 414 by masks and card). Few rows: by
// the reads of the cache. 64 tokens of 64 requests of 8k to 16k keys: 586 us, 5.5 TB/s.
// Measured and not kept: three tiles in LDS for the masked form (a whole step's time for each DMA,
// three workgroups a CU instead of four: 481 instead of 402 us); the same heads of every sequence on
// one XCD (no gain, 376 instead of 362 us where a group's keys were then read twice); a higher wave
// priority during the products (2% slower dense, 2% faster masked).
#include <type_traits>

#include "common.h"

#include "../../include/tasft_amd.h"

namespace tasft {

// A lambda called at several places is otherwise made a function, its captures in scratch memory.
#define TASFT_INLINE __attribute__((always_inline))

constexpr int kTile = 64;                // keys per tile
constexpr float kChunkMove = 8.f;        // a new maximum moves the exp2 reference only if this far above it
constexpr float kLn2 = 0.69314718055994531f;

struct ChunkParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* o;
  float* lse;  // [T, Hq] or null
  const uint8_t* mask;
  const int32_t* table;
  const int32_t* kv_lens;
  const int32_t* cu;
  float* ws_o;   // [T * Hq][P][D]
  float* ws_ml;  // [T * Hq][P][2]
  int64_t sq[2], so[2];  // (token, head)
  int64_t sk[3], sv[3];  // (page, token, head)
  int64_t sm[4];         // mask bytes (sequence, head, query block, key block)
  int64_t bt_stride;
  int N, T, Hq, Hkv, G, L;
  int ps_shift, num_pages, cap;  // cap: slots of the table
  int bs_shift, mask_rows;       // mask blocks of 1 << bs_shift tokens
  int QT, P;                     // row tiles per sequence and KV head (or head), key splits
  float scale_log2;
  int causal;
};

// A sequence's chunk: its first token, length, cached keys and first position. A length past the table
// (its keys are not there) leaves the tokens at the positions that the append gave them.
struct ChunkSeq {
  int t0, len, kv, p0;
};

__device__ __forceinline__ ChunkSeq chunk_seq(const ChunkParams& p, int n) {
  ChunkSeq s;
  s.t0 = min(max(p.cu[n], 0), p.T);
  const int t1 = min(max(p.cu[n + 1], s.t0), p.T);
  s.len = min(t1 - s.t0, p.L);
  const int full = max(p.kv_lens[n], 0);
  s.kv = min(full, p.cap);
  s.p0 = full - (t1 - s.t0);  // of the whole chunk, also where L cuts it
  return s;
}

// Rows of tokens behind the last sequence: 0 and -inf, shared out over the launch.
template <int D>
__device__ __forceinline__ void chunk_zero_tail(const ChunkParams& p, int64_t wg, int64_t wgs, int tid, int threads) {
  const int end = min(max(p.cu[p.N], 0), p.T);
  for (int64_t t = end + wg; t < p.T; t += wgs)
    for (int i = tid; i < p.Hq * (D / 8); i += threads) {
      const int h = i / (D / 8), c = i % (D / 8);
      *(u32x4_t*)(p.o + t * p.so[0] + h * p.so[1] + c * 8) = (u32x4_t){0u, 0u, 0u, 0u};
      if (c == 0 && p.lse) p.lse[t * p.Hq + h] = -INFINITY;
    }
}

// Rows of a KV head behind the first L tokens of a sequence: the join leaves out what has such a sum.
constexpr uint32_t kCutRow = 0xbf800000u;  // -1: no sum of exponentials
__device__ __forceinline__ void chunk_mark_cut(const ChunkParams& p, const ChunkSeq& s, int n, int kvh, int tid,
                                               int threads) {
  const int rows = (min(max(p.cu[n + 1], s.t0), p.T) - s.t0 - s.len) * p.G;
  for (int r = tid; r < rows; r += threads) {
    const int64_t t = s.t0 + s.len + r / p.G;
    p.ws_ml[((t * p.Hq + kvh * p.G + r % p.G) * p.P) * 2 + 1] = __uint_as_float(kCutRow);
  }
}

__device__ __forceinline__ void chunk_dma(__amdgpu_buffer_rsrc_t r, uint8_t* dst, int voff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (TASFT_LDS void*)dst, 16, voff, 0, 0, 0);
}

// The same of 4 bytes a lane.
__device__ __forceinline__ void chunk_dma4(__amdgpu_buffer_rsrc_t r, float* dst, int voff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (TASFT_LDS void*)dst, 4, voff, 0, 0, 0);
}

// s_waitcnt immediate: at most n vector memory operations outstanding.
constexpr int vm_wait(int n) { return (n & 15) | ((n >> 4) << 14) | (7 << 4) | (15 << 8); }

__device__ __forceinline__ void chunk_barrier() { asm volatile("s_barrier" ::: "memory"); }

// LDS position of 16-byte chunk cc of row r: K rows are read 32 at a time, V rows transposed.
template <int D>
__device__ __forceinline__ int chunk_swz_k(int r, int cc) {
  return cc ^ (D == 128 ? (r & 15) : ((r >> 1) & 7));
}
template <int D>
__device__ __forceinline__ int chunk_swz_v(int r, int cc) {
  return cc ^ (D == 128 ? ((r & 3) << 2) : (((r >> 1) & 1) << 2));
}

typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));

// A pair of 16-bit values with infinities and NaN replaced by 0.
template <int DT>
__device__ __forceinline__ uint32_t finite2(uint32_t w) {
  constexpr uint32_t E = DT == kF16 ? 0x7c00u : 0x7f80u;
  if ((w & E) == E) w &= 0xffff0000u;
  if ((w & (E << 16)) == (E << 16)) w &= 0xffffu;
  return w;
}

// A uniform 32-bit load from read-only memory through the scalar cache.
typedef const __attribute__((address_space(4))) int32_t* const_i32;
__device__ __forceinline__ int scalar_load(const int32_t* p) { return *(const_i32)(uintptr_t)p; }

// The kernel's argument read again: what only the end of a kernel uses is not kept in scalar
// registers over its main loop (they spilled).
typedef const __attribute__((address_space(4))) ChunkParams* ParamsPtr;
__device__ __forceinline__ ParamsPtr params_again() {
  ParamsPtr p = (ParamsPtr)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

constexpr int kRowTile = 128;  // rows of a dense workgroup: four waves
constexpr int kMaskTile = 64;  // positions of a masked one: two waves

// PIECES: runs of a wave's share of a tile that lie in one page each (one where pages are at least as
// long as the share). A template: the general form's scalar registers spilled, at a fifth of the time.
// MASK: kDense, kPositions (64 positions of a head), kRows (a mask, the dense form's rows).
enum ChunkMask { kDense = 0, kPositions = 1, kRows = 2 };
template <int D, int DT, int MASK, int PIECES>
__global__ void __launch_bounds__(MASK == kPositions ? 128 : 256)
    __attribute__((amdgpu_waves_per_eu(D == 64 && MASK == kPositions ? 3 : 2, D == 64 && MASK == kPositions ? 3 : 2)))
chunk_rows_kernel(const ChunkParams p) {
  constexpr bool MASKED = MASK == kPositions, ROWMASK = MASK == kRows;
  constexpr int WAVES = MASKED ? 2 : 4;
  constexpr int ROW_TILE = MASKED ? kMaskTile : kRowTile;
  static_assert(ROW_TILE == 32 * WAVES && (ROW_TILE & (ROW_TILE - 1)) == 0, "row tile");
  constexpr int KSTEPS = D / 16;
  constexpr int DTILES = D / 32;
  constexpr int ROWB = D * 2;
  constexpr int TILE = kTile * ROWB;
  constexpr int RPU = 1024 / ROWB;         // rows of a 1 KB DMA unit
  constexpr int WROWS = kTile / WAVES;     // rows of a tile that a wave brings
  constexpr int UPW = WROWS / RPU;         // its units
  constexpr int PROWS = WROWS / PIECES;
  static_assert(PROWS >= 8 && PROWS % RPU == 0, "a piece is whole units");
  __shared__ __attribute__((aligned(1024))) uint8_t k0_lds[TILE];
  __shared__ __attribute__((aligned(1024))) uint8_t v0_lds[TILE];
  __shared__ __attribute__((aligned(1024))) uint8_t k1_lds[MASKED ? 16 : TILE];
  __shared__ __attribute__((aligned(1024))) uint8_t v1_lds[MASKED ? 16 : TILE];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int grp16 = lane >> 4, t16 = lane & 15, tr_row = t16 >> 2, tr_cb = t16 & 3;

  chunk_zero_tail<D>(p, blockIdx.x, gridDim.x, tid, WAVES * kWave);

  // The (sequence, KV head) whose K and V the workgroup reads, and its place among those that do:
  // one XCD's L2 serves them all.
  const int members = p.QT * (MASKED ? p.G : 1) * p.P;
  int64_t group;
  int member;
  xcd_group_map(blockIdx.x, (int64_t)p.N * p.Hkv, members, &group, &member);
  const int n = (int)(group / p.Hkv), kvh = (int)(group % p.Hkv);
  const int split = member % p.P;
  member /= p.P;
  // The longest rows first, of all heads: the short ones fill the launch's end (a prompt of 8192
  // tokens 574 us in order, 513 so; masked 315 and 290).
  const int gm = MASKED ? member % p.G : 0, qt = p.QT - 1 - (MASKED ? member / p.G : member);
  const ChunkSeq sq = chunk_seq(p, n);
  if (sq.len == 0) return;
  if (p.P > 1 && split == 0 && qt == 0 && gm == 0) chunk_mark_cut(p, sq, n, kvh, tid, WAVES * kWave);

  // This lane's row (token i of the chunk, head h), the wave's range of tokens and the workgroup's
  // last token.
  int i, h, i_first, i_last, i_end;
  bool row_ok;
  if constexpr (MASKED) {
    // Positions aligned to the row tile: a wave's 32 rows lie in one mask block.
    const int base = qt * ROW_TILE - (sq.p0 & (ROW_TILE - 1));
    if (base >= sq.len) return;
    i_first = max(base + wave * 32, 0);
    i_last = min(base + wave * 32 + 31, sq.len - 1);
    i_end = min(base + ROW_TILE, sq.len) - 1;
    i = base + wave * 32 + col;
    h = kvh * p.G + gm;
    row_ok = i >= 0 && i < sq.len;
  } else {
    const int rows = sq.len * p.G, r0 = qt * ROW_TILE;
    if (r0 >= rows) return;
    const int rw = r0 + wave * 32, r = rw + col;
    i = r / p.G;
    h = kvh * p.G + (r - i * p.G);
    row_ok = r < rows;
    i_first = rw / p.G;
    i_last = rw < rows ? min(rw + 31, rows - 1) / p.G : -1;
    i_end = (min(r0 + ROW_TILE, rows) - 1) / p.G;
  }
  const bool wave_on = i_first <= i_last;
  if (!row_ok) {  // reads a row of the chunk, is not stored
    i = min(max(i, 0), sq.len - 1);
    h = kvh * p.G;
  }
  // Keys a row sees: 0 .. lim. All rows of the wave see the keys to all_see, none one past any_see.
  const int lim = p.causal ? min(sq.p0 + i, sq.kv - 1) : sq.kv - 1;
  const int all_see = p.causal ? min(sq.p0 + i_first, sq.kv - 1) : sq.kv - 1;
  const int any_see = !wave_on ? -1 : (p.causal ? min(sq.p0 + i_last, sq.kv - 1) : sq.kv - 1);
  const int wg_see = p.causal ? min(sq.p0 + i_end, sq.kv - 1) : sq.kv - 1;
  const int tiles = wg_see < 0 ? 0 : wg_see / kTile + 1;
  const int tile_a = (int)((int64_t)split * tiles / p.P), tile_b = (int)((int64_t)(split + 1) * tiles / p.P);

  // Q as the B operand, lane (col, half): dims 16 ks + 8 half .. + 7 of its row.
  u32x4_t qf[KSTEPS];
  {
    const uint16_t* qr = p.q + (int64_t)(sq.t0 + i) * p.sq[0] + h * p.sq[1] + half * 8;
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks) qf[ks] = *(const u32x4_t*)(qr + ks * 16);
  }

  // The tiles of the split in order; masked: those that any row's block mask selects, with this
  // wave's own two bits (the 32-key halves, which differ at mask blocks of 32 only).
  int cursor = tile_a, chunk = tile_a - kWave, own_next = 0;
  uint64_t ubits = 0, own0 = 0, own1 = 0;
  const uint8_t* mseq = nullptr;
  int row_lo = 0, row_hi = 0, row_own = 0;  // mask rows; row_own: the wave's (positions), the lane's (rows)
  if constexpr (ROWMASK) {
    mseq = p.mask + n * p.sm[0] + (int64_t)kvh * p.G * p.sm[1];
    const int block0 = sq.p0 >> p.bs_shift;
    auto row_of = [&](int j) { return min(max(((sq.p0 + j) >> p.bs_shift) - block0, 0), p.mask_rows - 1); };
    row_lo = row_of(0);
    row_hi = row_of(i_end);
    row_own = row_of(i);
  }
  if constexpr (MASKED) {
    mseq = p.mask + n * p.sm[0] + (int64_t)(kvh * p.G + gm) * p.sm[1];
    const int block0 = sq.p0 >> p.bs_shift;
    auto row_of = [&](int j) { return min(max(((sq.p0 + j) >> p.bs_shift) - block0, 0), p.mask_rows - 1); };
    row_lo = row_of(max(qt * ROW_TILE - (sq.p0 & (ROW_TILE - 1)), 0));
    row_hi = row_of(i_end);
    row_own = wave_on ? row_of(i_first) : -1;
  }
  auto next_tile = [&]() TASFT_INLINE -> int {
    if constexpr (MASK == kDense) {
      return cursor < tile_b ? cursor++ : -1;
    } else if constexpr (ROWMASK) {
      while (ubits == 0) {
        chunk += kWave;
        if (chunk >= tile_b) return -1;
        const int kt = min(chunk + lane, tile_b - 1);
        const int b0 = p.bs_shift == 5 ? 2 * kt : kt >> (p.bs_shift - 6);
        const int b1 = p.bs_shift == 5 ? min(2 * kt + 1, (p.cap - 1) >> 5) : b0;
        // Every head's rows of the mask, four heads' loads in flight; a lane keeps its own row's.
        uint32_t any = 0;
        own0 = own1 = 0;
        for (int g0 = 0; g0 < p.G; g0 += 4)
          for (int r = row_lo; r <= row_hi; ++r) {
            uint32_t x[4], y[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const uint8_t* m = mseq + min(g0 + g, p.G - 1) * p.sm[1] + r * p.sm[2];
              x[g] = m[b0 * p.sm[3]];
              y[g] = m[b1 * p.sm[3]];
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const bool mine = h - kvh * p.G == g0 + g && row_own == r;
              const uint64_t bx = __ballot(x[g] != 0), by = __ballot(y[g] != 0);
              own0 = mine ? bx : own0;
              own1 = mine ? by : own1;
              any |= x[g] | y[g];
            }
          }
        ubits = __ballot(any != 0 && chunk + lane < tile_b);
      }
      const int b = __builtin_ctzll(ubits);
      ubits &= ubits - 1;
      own_next = (int)((own0 >> b) & 1) | (int)((own1 >> b) & 1) << 1;
      return chunk + b;
    } else {
      while (ubits == 0) {
        chunk += kWave;
        if (chunk >= tile_b) return -1;
        const int kt = min(chunk + lane, tile_b - 1);
        const int b0 = p.bs_shift == 5 ? 2 * kt : kt >> (p.bs_shift - 6);
        const int b1 = p.bs_shift == 5 ? min(2 * kt + 1, (p.cap - 1) >> 5) : b0;
        uint32_t any = 0, mine0 = 0, mine1 = 0;
        for (int r = row_lo; r <= row_hi; ++r) {
          const uint32_t x = mseq[r * p.sm[2] + b0 * p.sm[3]], y = mseq[r * p.sm[2] + b1 * p.sm[3]];
          any |= x | y;
          if (r == row_own) mine0 = x, mine1 = y;
        }
        ubits = __ballot(any != 0 && chunk + lane < tile_b);
        own0 = __ballot(mine0 != 0);
        own1 = __ballot(mine1 != 0);
      }
      const int b = __builtin_ctzll(ubits);
      ubits &= ubits - 1;
      own_next = (int)((own0 >> b) & 1) | (int)((own1 >> b) & 1) << 1;
      return chunk + b;
    }
  };

  // A wave brings rows WROWS wave .. of a tile, PROWS from a page. A buffer resource ends with the
  // last row below kv_len: rows past it arrive as zeros. Per-lane source offsets, from the wave's
  // first row: the lane loads the chunk that the self-inverse swizzle maps to its 16 bytes.
  const uint16_t* kbase = p.k + kvh * p.sk[2];
  const uint16_t* vbase = p.v + kvh * p.sv[2];
  const int32_t* table = p.table + n * p.bt_stride;
  int koff[UPW], voff[UPW];
#pragma unroll
  for (int u = 0; u < UPW; ++u) {
    const int row = u * RPU + lane / (ROWB / 16), pos = lane % (ROWB / 16);
    koff[u] = (row * (int)p.sk[1] + chunk_swz_k<D>(row, pos) * 8) * 2;
    voff[u] = (row * (int)p.sv[1] + chunk_swz_v<D>(row, pos) * 8) * 2;
  }
  struct Pages {
    int id[PIECES];
  };
  auto load_pages = [&](int kt) TASFT_INLINE -> Pages {
    const int r = kt * kTile + wave * WROWS, last = (sq.kv - 1) >> p.ps_shift;
    Pages pg;
#pragma unroll
    for (int e = 0; e < PIECES; ++e) pg.id[e] = scalar_load(table + min((r + PROWS * e) >> p.ps_shift, last));
    return pg;
  };
  // The wave's share of a tile of K or V: base of the head's pool, its page and token strides.
  auto dma_rows = [&](uint8_t* tile_lds, const uint16_t* base, int64_t page_st, int tok_st, const int* off, int kt,
                      const Pages& pg) TASFT_INLINE {
    const int r = kt * kTile + wave * WROWS, left = sq.kv - r;
#pragma unroll
    for (int e = 0; e < PIECES; ++e) {
      // A later piece's resource starts PROWS e rows before it: offsets count from the wave's first.
      const int in_page = ((r + PROWS * e) & ((1 << p.ps_shift) - 1)) - PROWS * e;
      const uint16_t* from = base + min(max(pg.id[e], 0), p.num_pages - 1) * page_st + (int64_t)in_page * tok_st;
      const int rows = min(left, PROWS * (e + 1));
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          (void*)from, (short)0, left > PROWS * e ? (rows - 1) * tok_st * 2 + ROWB : 0, 0x00020000);
#pragma unroll
      for (int u = e * (PROWS / RPU); u < (e + 1) * (PROWS / RPU); ++u)
        chunk_dma(rs, tile_lds + (wave * UPW + u) * 1024, off[u]);
    }
  };
  auto dma_k = [&](uint8_t* tile_lds, int kt, const Pages& pg) TASFT_INLINE {
    dma_rows(tile_lds, kbase, p.sk[0], (int)p.sk[1], koff, kt, pg);
  };
  auto dma_v = [&](uint8_t* tile_lds, int kt, const Pages& pg) TASFT_INLINE {
    dma_rows(tile_lds, vbase, p.sv[0], (int)p.sv[1], voff, kt, pg);
  };

  f32x16_t oacc[DTILES];
#pragma unroll
  for (int dt = 0; dt < DTILES; ++dt) oacc[dt] = (f32x16_t){};
  float m_ref = -INFINITY;  // exp2 reference of this lane's row (log2 domain)
  float l_run = 0.f;
  int fix_from = 0x7fffffff;  // first tile whose infinities or NaN of V were left out

  // Whether this wave has anything to do with a tile.
  auto takes_part = [&](int kt, int own) {
    if constexpr (ROWMASK) return kt * kTile <= any_see && __ballot(row_ok && own != 0) != 0;
    return kt * kTile <= any_see && (!MASKED || own != 0);
  };
  // S^T of a tile. Register rr of s0 / s1 is key 4 half + off(rr) (+ 32), off = 8 (rr / 4) + rr % 4.
  auto scores = [&](const uint8_t* kS, f32x16_t& s0, f32x16_t& s1) TASFT_INLINE {
    u32x4_t kf[2][KSTEPS];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks) {
        const int r = t * 32 + col;
        kf[t][ks] = *(const u32x4_t*)(kS + r * ROWB + chunk_swz_k<D>(r, ks * 2 + half) * 16);
      }
    s0 = s1 = (f32x16_t){};
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks) {
      s0 = mfma16<DT>(kf[0][ks], qf[ks], s0);
      s1 = mfma16<DT>(kf[1][ks], qf[ks], s1);
    }
  };
  // Whether some row of the wave does not see some key of the tile.
  auto is_mixed = [&](int kt, int own) {
    if constexpr (ROWMASK) return kt * kTile + kTile - 1 > all_see || __ballot(own != 3) != 0;
    return kt * kTile + kTile - 1 > all_see || (MASKED && own != 3);
  };
  // The softmax step: P^T as the B operand of the second product.
  auto softmax = [&](f32x16_t& s0, f32x16_t& s1, int kt, int own, bool mixed, u32x4_t (&pb)[4]) TASFT_INLINE {
    const int key0 = kt * kTile;
    const int lim0 = MASK != kDense && !(own & 1) ? -1 : lim - key0 - 4 * half;
    const int lim1 = MASK != kDense && !(own & 2) ? -1 : lim - key0 - 4 * half - 32;
    if (mixed) {
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
    const float mloc = pair_max32(fmaxf(fmaxf(ma, s0[15]), fmaxf(mb, s1[15]))) * p.scale_log2;
    const bool move = mloc > m_ref + kChunkMove;
    if (__ballot(move)) {
      const float alpha = move ? __builtin_amdgcn_exp2f(m_ref - mloc) : 1.f;
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < DTILES; ++dt) oacc[dt] *= alpha;
      m_ref = move ? mloc : m_ref;
    }
    const float m_use = (m_ref == -INFINITY) ? 0.f : m_ref;
    float lsum0 = 0.f, lsum1 = 0.f;
#pragma unroll
    for (int rr = 0; rr < 16; ++rr) {
      const float e0 = __builtin_amdgcn_exp2f(fmaf(s0[rr], p.scale_log2, -m_use));
      const float e1 = __builtin_amdgcn_exp2f(fmaf(s1[rr], p.scale_log2, -m_use));
      s0[rr] = e0;
      s1[rr] = e1;
      lsum0 += e0;
      lsum1 += e1;
    }
    l_run += lsum0 + lsum1;
#pragma unroll
    for (int pp = 0; pp < 4; ++pp) {
      const f32x16_t& sv = (pp < 2) ? s0 : s1;
      const int o = 8 * (pp & 1);
      pb[pp] = (u32x4_t){pack16x2<DT>(sv[o + 0], sv[o + 1]), pack16x2<DT>(sv[o + 2], sv[o + 3]),
                         pack16x2<DT>(sv[o + 4], sv[o + 5]), pack16x2<DT>(sv[o + 6], sv[o + 7])};
    }
  };
  // O^T += V^T P^T.
  auto add_values = [&](const uint8_t* vS, int kt, bool mixed, const u32x4_t (&pb)[4]) TASFT_INLINE {
    u32x2_t vlo[4][DTILES], vhi[4][DTILES];
#pragma unroll
    for (int pp = 0; pp < 4; ++pp) {
      const int kk = 16 * pp + 4 * (grp16 >> 1);
#pragma unroll
      for (int dt = 0; dt < DTILES; ++dt) {
        const int d0 = dt * 32 + 16 * (grp16 & 1) + 4 * tr_cb;
        const int cc = d0 >> 3, sub = (d0 & 7) * 2;
        const int r1 = kk + tr_row, r2 = r1 + 8;
        vlo[pp][dt] = ds_read_tr16_b64((const void*)(vS + r1 * ROWB + chunk_swz_v<D>(r1, cc) * 16 + sub));
        vhi[pp][dt] = ds_read_tr16_b64((const void*)(vS + r2 * ROWB + chunk_swz_v<D>(r2, cc) * 16 + sub));
      }
    }
    if (mixed) {
      // The largest magnitudes tell whether there is one (two instructions a pair of values).
      u16x2_t top = {0, 0};
#pragma unroll
      for (int pp = 0; pp < 4; ++pp)
#pragma unroll
        for (int dt = 0; dt < DTILES; ++dt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, vlo[pp][dt][j] & 0x7fff7fffu));
            top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, vhi[pp][dt][j] & 0x7fff7fffu));
          }
      constexpr uint16_t E = DT == kF16 ? 0x7c00 : 0x7f80;
      if (__ballot(top[0] >= E || top[1] >= E)) {
        fix_from = min(fix_from, kt);
#pragma unroll
        for (int pp = 0; pp < 4; ++pp)
#pragma unroll
          for (int dt = 0; dt < DTILES; ++dt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              vlo[pp][dt][j] = finite2<DT>(vlo[pp][dt][j]);
              vhi[pp][dt][j] = finite2<DT>(vhi[pp][dt][j]);
            }
      }
    }
#pragma unroll
    for (int pp = 0; pp < 4; ++pp)
#pragma unroll
      for (int dt = 0; dt < DTILES; ++dt) {
        const u32x4_t a = {vlo[pp][dt][0], vlo[pp][dt][1], vhi[pp][dt][0], vhi[pp][dt][1]};
        oacc[dt] = mfma16<DT>(a, pb[pp], oacc[dt]);
      }
  };

  int cur = next_tile(), own_cur = own_next;
  if constexpr (!MASKED) {
    int nxt = -1, own_nxt = 0;
    Pages pg = {};
    if (cur >= 0) {
      const Pages first = load_pages(cur);
      dma_k(k0_lds, cur, first);
      dma_v(v0_lds, cur, first);
      nxt = next_tile();
      own_nxt = own_next;
      if (nxt >= 0) pg = load_pages(nxt);
    }
    // One tile from a stage while the next one's DMA fills the other: by the barrier every wave's
    // share of this tile has landed and every wave is done with the tile before it.
    auto step = [&](uint8_t* ka, uint8_t* va, uint8_t* kb, uint8_t* vb) TASFT_INLINE {
      __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
      chunk_barrier();
      int nn = -1, own_nn = 0;
      Pages pn = pg;
      if (nxt >= 0) {
        dma_k(kb, nxt, pg);
        dma_v(vb, nxt, pg);
        nn = next_tile();
        own_nn = own_next;
        if (nn >= 0) pn = load_pages(nn);
      }
      const int own = ROWMASK ? own_cur : 3;
      if (takes_part(cur, own)) {
        const bool mixed = is_mixed(cur, own);
        f32x16_t s0, s1;
        u32x4_t pb[4];
        scores(ka, s0, s1);
        softmax(s0, s1, cur, own, mixed, pb);
        add_values(va, cur, mixed, pb);
      }
      cur = nxt;
      own_cur = own_nxt;
      nxt = nn;
      own_nxt = own_nn;
      pg = pn;
    };
    while (cur >= 0) {
      step(k0_lds, v0_lds, k1_lds, v1_lds);
      if (cur < 0) break;
      step(k1_lds, v1_lds, k0_lds, v0_lds);
    }
  } else {
    // One K and one V tile, four workgroups a CU (three waves per SIMD at D = 64): the V DMA starts
    // once every wave is done with the V tile, the next K's once every wave has read this K.
    constexpr int kWaitTile = vm_wait(UPW);  // all but the last tile's units have landed
    Pages pg = {};
    if (cur >= 0) {
      pg = load_pages(cur);
      dma_k(k0_lds, cur, pg);
    }
    while (cur >= 0) {
      __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0): own share of K landed, V's reads returned
      chunk_barrier();
      dma_v(v0_lds, cur, pg);
      const bool on = takes_part(cur, own_cur), mixed = is_mixed(cur, own_cur);
      f32x16_t s0 = (f32x16_t){}, s1 = (f32x16_t){};
      u32x4_t pb[4] = {};
      if (on) scores(k0_lds, s0, s1);
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this wave's K reads returned
      chunk_barrier();                     // every wave has read K
      const int nxt = next_tile(), own_nxt = own_next;
      // Always one K tile after V (the last one again at the end), so that V's wait is one count.
      const Pages pn = load_pages(nxt >= 0 ? nxt : cur);
      dma_k(k0_lds, nxt >= 0 ? nxt : cur, pn);
      if (on) softmax(s0, s1, cur, own_cur, mixed, pb);
      __builtin_amdgcn_s_waitcnt(kWaitTile);  // own share of V landed, the next K in flight
      chunk_barrier();
      if (on) add_values(v0_lds, cur, mixed, pb);
      cur = nxt;
      own_cur = own_nxt;
      pg = pn;
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);  // no DMA into this workgroup's LDS outlives it
  }

  const ParamsPtr pe = params_again();
  if (fix_from != 0x7fffffff) {
    // Infinities and NaN of V in tiles that only some of the wave's rows see: key by key, from
    // memory, to the rows that see the key. (Where a later tile had them in its product, once
    // more changes nothing.)
    const float m_use = (m_ref == -INFINITY) ? 0.f : m_ref;
    const int last = min(any_see, tile_b * kTile - 1);
#pragma nounroll
    for (int key = fix_from * kTile; key <= last; ++key) {
      const int64_t page = min(max(pe->table[n * pe->bt_stride + (key >> pe->ps_shift)], 0), pe->num_pages - 1);
      const int in_page = key & ((1 << pe->ps_shift) - 1);
      const uint16_t* vr = pe->v + kvh * pe->sv[2] + page * pe->sv[0] + in_page * pe->sv[1];
      const uint32_t w = *(const uint32_t*)(vr + (lane * 2) % D);
      if (!__ballot(finite2<DT>(w) != w)) continue;
      bool sees = row_ok && key <= lim;
      if constexpr (MASK != kDense) {
        const int head = MASKED ? kvh * pe->G + gm : h;
        const uint8_t* m = pe->mask + n * pe->sm[0] + (int64_t)head * pe->sm[1] + row_own * pe->sm[2];
        sees = sees && m[(key >> pe->bs_shift) * pe->sm[3]] != 0;
      }
      const uint16_t* kr = pe->k + kvh * pe->sk[2] + page * pe->sk[0] + in_page * pe->sk[1] + half * 8;
      float dot = 0.f;
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks) {
        float x[8], y[8];
        unpack16x8<DT>(*(const u32x4_t*)(kr + ks * 16), x);
        unpack16x8<DT>(qf[ks], y);
#pragma unroll
        for (int j = 0; j < 8; ++j) dot = fmaf(x[j], y[j], dot);
      }
      const float pk = __builtin_amdgcn_exp2f(fmaf(pair_sum32(dot), pe->scale_log2, -m_use));
#pragma unroll
      for (int dt = 0; dt < DTILES; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint32_t x = vr[dt * 32 + 8 * (e >> 2) + 4 * half + (e & 3)];
          const bool add = sees & (finite2<DT>(x) != x);
          oacc[dt][e] += add ? pk * bits16_to_f32<DT>(x) : 0.f;
        }
    }
  }

  const float l_tot = pair_sum32(l_run);
  const int64_t tok = sq.t0 + i;
  if (pe->P > 1) {
    const int64_t row = (tok * pe->Hq + h) * pe->P + split;
    if (row_ok) {
      if (half == 0) {
        pe->ws_ml[row * 2] = m_ref;
        pe->ws_ml[row * 2 + 1] = l_tot;
      }
      float* wo = pe->ws_o + row * D;
#pragma unroll
      for (int dt = 0; dt < DTILES; ++dt)
#pragma unroll
        for (int gq = 0; gq < 4; ++gq)
          *(f32x4_t*)(wo + dt * 32 + 8 * gq + 4 * half) =
              (f32x4_t){oacc[dt][4 * gq], oacc[dt][4 * gq + 1], oacc[dt][4 * gq + 2], oacc[dt][4 * gq + 3]};
    }
    return;
  }
  if (pe->lse && row_ok && half == 0) pe->lse[tok * pe->Hq + h] = (m_ref + __builtin_amdgcn_logf(l_tot)) * kLn2;
  const float inv = 1.f / (l_tot > 0.f ? l_tot : 1.f);  // empty rows: 0; NaN rows stay NaN
  // Whole rows through LDS: 16-byte chunk c of row r at position c ^ (r % chunks).
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  chunk_barrier();                     // every wave is done with the tiles
  uint8_t* ost = ((wave & 2) ? v0_lds : k0_lds) + (wave & 1) * (32 * ROWB);
  constexpr int CPR = ROWB / 16;
#pragma unroll
  for (int dt = 0; dt < DTILES; ++dt)
#pragma unroll
    for (int gq = 0; gq < 4; ++gq) {
      const int d0 = dt * 32 + 8 * gq + 4 * half;
      const u32x2_t w = {pack16x2<DT>(oacc[dt][4 * gq + 0] * inv, oacc[dt][4 * gq + 1] * inv),
                         pack16x2<DT>(oacc[dt][4 * gq + 2] * inv, oacc[dt][4 * gq + 3] * inv)};
      *(u32x2_t*)(ost + col * ROWB + (((d0 >> 3) ^ (col & (CPR - 1))) << 4) + (d0 & 7) * 2) = w;
    }
  const int64_t at = row_ok ? tok * pe->so[0] + h * pe->so[1] : -1;
#pragma unroll
  for (int j = 0; j < 32 * CPR / kWave; ++j) {
    const int r = j * (kWave / CPR) + lane / CPR, c = lane % CPR;
    const u32x4_t x = *(const u32x4_t*)(ost + r * ROWB + ((c ^ (r & (CPR - 1))) << 4));
    const int64_t to = __shfl(at, r, kWave);
    if (to >= 0) *(u32x4_t*)(pe->o + to + c * 8) = x;
  }
}

// Joins the P splits of every row; the partial sums of splits that saw no key are not used (they may
// be unwritten). Up to kFewSplits: D / 4 lanes a row, every split's loads in flight together. More:
// a workgroup a row, its factors computed once, the splits shared out over groups of D / 4 lanes,
// four loads in flight each (one lane walking 64 splits took 34 us for 32 rows, this 6).
constexpr int kFewSplits = 8;

template <int D, int DT>
__device__ __forceinline__ void chunk_store(const ChunkParams& p, int64_t row, int c, const f32x4_t& O, float L,
                                            float M) {
  const int64_t t = row / p.Hq;
  const int h = (int)(row - t * p.Hq);
  const float inv = 1.f / (L > 0.f ? L : 1.f);
  const u32x2_t w = {pack16x2<DT>(O[0] * inv, O[1] * inv), pack16x2<DT>(O[2] * inv, O[3] * inv)};
  *(u32x2_t*)(p.o + t * p.so[0] + h * p.so[1] + c * 4) = w;
  if (p.lse && c == 0) p.lse[row] = (M + __builtin_amdgcn_logf(L)) * kLn2;
}

template <int D, int DT>
__global__ void __launch_bounds__(256) chunk_combine_few_kernel(const ChunkParams p) {
  constexpr int LPR = D / 4;
  const int64_t row = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const int c = threadIdx.x % LPR;
  if (row >= (int64_t)min(max(p.cu[p.N], 0), p.T) * p.Hq) return;
  const float* ml = p.ws_ml + row * p.P * 2;
  const float* os = p.ws_o + row * p.P * D + c * 4;
  float m[kFewSplits], l[kFewSplits];
  f32x4_t o[kFewSplits];
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {  // past the last split: it again, not used
    const int at = min(s, p.P - 1);
    m[s] = ml[2 * at];
    l[s] = ml[2 * at + 1];
    o[s] = *(const f32x4_t*)(os + (int64_t)at * D);
  }
  if (__float_as_uint(l[0]) == kCutRow) return;  // behind the loads: not one more wait before them
  float M = -INFINITY;
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) M = fmaxf(M, m[s]);
  const float Mu = (M == -INFINITY) ? 0.f : M;
  float L = 0.f;
  f32x4_t O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s)
    if (s < p.P && __float_as_uint(l[s]) != 0u) {
      const float f = __builtin_amdgcn_exp2f(m[s] - Mu);
      L += l[s] * f;
      O += o[s] * f;
    }
  chunk_store<D, DT>(p, row, c, O, L, M);
}

template <int D, int DT>
__global__ void __launch_bounds__(256) chunk_combine_kernel(const ChunkParams p) {
  constexpr int LPR = D / 4, GROUPS = 256 / LPR;
  __shared__ float fac[1024];
  __shared__ float red[2][4];
  __shared__ f32x4_t part[GROUPS][LPR];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = tid % LPR, grp = tid / LPR;
  if (row >= (int64_t)min(max(p.cu[p.N], 0), p.T) * p.Hq) return;
  const float* ml = p.ws_ml + row * p.P * 2;
  const bool cut = __float_as_uint(ml[1]) == kCutRow;
  const float* os = p.ws_o + row * p.P * D + c * 4;
  float M = -INFINITY;
  for (int s = tid; s < p.P; s += 256) M = fmaxf(M, ml[2 * s]);
  M = wave_max(M);
  if (lane == 0) red[0][wave] = M;
  __syncthreads();
  M = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  const float Mu = (M == -INFINITY) ? 0.f : M;
  float L = 0.f;
  for (int s = tid; s < p.P; s += 256) {
    const float l = ml[2 * s + 1];
    const bool none = __float_as_uint(l) == 0u;
    const float f = none ? -1.f : __builtin_amdgcn_exp2f(ml[2 * s] - Mu);  // -1: not used
    fac[s] = f;
    L += none ? 0.f : l * f;
  }
  L = wave_sum(L);
  if (lane == 0) red[1][wave] = L;
  __syncthreads();
  L = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  f32x4_t O = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = grp; s0 < p.P; s0 += 4 * GROUPS) {
    f32x4_t x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *(const f32x4_t*)(os + (int64_t)min(s0 + i * GROUPS, p.P - 1) * D);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = s0 + i * GROUPS;
      const float f = s < p.P ? fac[s] : -1.f;
      if (__float_as_uint(f) != 0xbf800000u) O += x[i] * f;
    }
  }
  part[grp][c] = O;
  __syncthreads();
  if (grp != 0 || cut) return;
#pragma unroll
  for (int g = 1; g < GROUPS; ++g) O += part[g][c];
  chunk_store<D, DT>(p, row, c, O, L, M);
}

// ---------------------------------------------------------------------------------------
// Accumulated key weights: out[n, g, j] = in[n, g, j] + sum over the chunk's rows that see key j
// of exp(q . k_j scale - lse). The transpose of the attention's reduction: a wave keeps 64 keys
// (their K in registers as the A operand) and walks the rows 32 at a time (Q as the B operand),
// adding exp2 of the scores to one register per key; lanes are summed once at the end. Fixed
// order, no atomics.
//
// KW of the waves hold different keys, the others share out the rows of the same. Many keys (KW = 4
// of 4 waves) read Q less often, few keys (KW = 1) want four times as many workgroups. Where there
// are many rows (RING) they come by DMA through LDS: as loads into a lane's registers the rows'
// pieces of 16 bytes touch a line each, and the first-level cache bounds the kernel. KW = 4 walks the
// same rows with all waves, 64 a step, in a ring of four stages filled three steps ahead (a step is
// shorter than a trip to L2); KW = 1 gives each of eight waves two stages of 32 rows of its own,
// without a barrier. With few rows each wave loads its own into registers, the next tile's under
// the exponentials of one.
//
// Many rows: 32 rows and 64 keys are 512 cycles of products and 768 of exponentials, multiply-adds and
// sums, on two waves per SIMD, of which one's products hardly run beside the other's exponentials: 256
// tokens of 2 requests over 28k keys on average take 125 us (0.84 PFLOP/s, 34% MFMA busy), one after the
// other they would take 105. Few rows: by the reads of K (one token of 32 requests over 4097 keys,
// 28 / 4 heads: 28.5 us, 4.9 TB/s).
// ---------------------------------------------------------------------------------------
struct WeightParams {
  ChunkParams c;
  const float* scores;  // [N, Hkv, cap] (element strides ss) or null
  int64_t ss[3];
  float* out;           // [N, Hkv, cap] contiguous
  const float* lse;     // [T, Hq], strides (token, head)
  int64_t sl[2];
};

// A lane's place among the rows of a KV head (token i of the chunk, query head g of the group),
// moved a fixed number of rows at a time without a division.
struct RowPlace {
  int i, g;
  __device__ __forceinline__ void move(int di, int dg, int G) {
    i += di;
    g += dg;
    if (g >= G) {
      g -= G;
      ++i;
    }
  }
};

constexpr int weight_waves(int kw, bool ring) { return kw == 1 && ring ? 8 : 4; }

template <int D, int DT, int KW, bool RING, bool MASKED>
__global__ void __launch_bounds__(weight_waves(KW, RING) * kWave)
    __attribute__((amdgpu_waves_per_eu(RING && (D == 128 || KW == 1) ? 2 : 3)))
chunk_weights_kernel(const WeightParams wp) {
  constexpr int KSTEPS = D / 16;
  constexpr int ROWB = D * 2;
  constexpr int RPU = 1024 / ROWB;
  constexpr int WAVES = weight_waves(KW, RING);
  constexpr int RW = WAVES / KW;           // waves that share one of the KW sets of keys
  constexpr bool OWN = RING && KW == 1;    // two stages of its own for every wave
  constexpr int STAGE = OWN ? WAVES * 32 * ROWB : RING ? kTile * ROWB : 16;
  const ChunkParams& p = wp.c;
  __shared__ __attribute__((aligned(1024))) uint8_t s0_lds[STAGE];
  __shared__ __attribute__((aligned(1024))) uint8_t s1_lds[STAGE];
  __shared__ __attribute__((aligned(1024))) uint8_t s2_lds[OWN ? 16 : STAGE];
  __shared__ __attribute__((aligned(1024))) uint8_t s3_lds[OWN ? 16 : STAGE];
  __shared__ float lse_lds[4][WAVES][kWave];   // stage, wave (its own copy), row; few keys: the sums
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kg = wave % KW, rg = wave / KW;
  const int col = lane & 31, half = lane >> 5;
  const int per = (p.cap + KW * kTile - 1) / (KW * kTile);  // workgroups per (sequence, KV head)
  int64_t group;
  int member;
  xcd_group_map(blockIdx.x, (int64_t)p.N * p.Hkv, per, &group, &member);
  const int n = (int)(group / p.Hkv), kvh = (int)(group % p.Hkv);
  const ChunkSeq sq = chunk_seq(p, n);
  const int key0 = (member * KW + kg) * kTile;
  const int wg0 = member * KW * kTile;

  float total = 0.f;  // of this lane's key, in the first wave of its keys
  if (wg0 < sq.kv && sq.len > 0) {
    // K as the A operand, from memory: keys 32 t + col, dims 16 ks + 8 half .. + 7. (Once per wave;
    // through LDS it took the memory of another workgroup per CU.) Keys past the last one read it.
    u32x4_t kf[2][KSTEPS];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int r = min(key0 + t * 32 + col, sq.kv - 1);
      const int64_t page = min(max(p.table[n * p.bt_stride + (r >> p.ps_shift)], 0), p.num_pages - 1);
      const uint16_t* kr = p.k + page * p.sk[0] + (r & ((1 << p.ps_shift) - 1)) * p.sk[1] + kvh * p.sk[2] + half * 8;
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks) kf[t][ks] = *(const u32x4_t*)(kr + ks * 16);
    }
    f32x16_t a0 = (f32x16_t){}, a1 = (f32x16_t){};
    const int rows = sq.len * p.G;
    // The first row that sees the workgroup's first key.
    const int first = p.causal ? max(wg0 - sq.p0, 0) : 0;
    const int block0 = sq.p0 >> (MASKED ? p.bs_shift : 0);
    const int r_first = (int)min((int64_t)first * p.G, (int64_t)rows);

    // Adds a tile of 32 rows: Q as the B operand; this lane's row is at `at`, its log-sum `lse`.
    // between() runs when Q has been used.
    auto add_rows = [&](const u32x4_t* qf, RowPlace at, bool ok, float lse, auto between) TASFT_INLINE {
      const int pos = (int)((uint32_t)sq.p0 + (uint32_t)at.i);  // of a row past the last one any number
      const int lim = p.causal ? min(pos, sq.kv - 1) : sq.kv - 1;
      // How far the row sees into the two halves of the keys, in the lane's count. A row without
      // keys (lse -inf) or behind the last one adds nothing.
      int lim0 = ok && lse != -INFINITY ? lim - key0 - 4 * half : -1, lim1 = lim0 - 32;
      if constexpr (MASKED) {
        // (A row past the last one stays within the mask, by its row's and head's limits.)
        const int mr = min(max((pos >> p.bs_shift) - block0, 0), p.mask_rows - 1);
        const uint8_t* m = p.mask + n * p.sm[0] + (int64_t)(kvh * p.G + at.g) * p.sm[1] + mr * p.sm[2];
        const int last_block = (p.cap - 1) >> p.bs_shift;
        if (m[min(key0 >> p.bs_shift, last_block) * p.sm[3]] == 0) lim0 = -1;
        if (m[min((key0 + 32) >> p.bs_shift, last_block) * p.sm[3]] == 0) lim1 = -1;
      }
      // Many tiles: those that no row sees are left out, and the selections of those that all see.
      if (RING && __ballot(max(lim0, lim1) >= 0) == 0) return;
      f32x16_t s0 = (f32x16_t){}, s1 = (f32x16_t){};
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks) {
        s0 = mfma16<DT>(kf[0][ks], qf[ks], s0);
        s1 = mfma16<DT>(kf[1][ks], qf[ks], s1);
      }
      between();
      const float l2 = lse * kLog2e;
#pragma unroll
      for (int rr = 0; rr < 16; ++rr) {
        s0[rr] = __builtin_amdgcn_exp2f(fmaf(s0[rr], p.scale_log2, -l2));
        s1[rr] = __builtin_amdgcn_exp2f(fmaf(s1[rr], p.scale_log2, -l2));
      }
      // The last key of a half has offset 27 in the lanes' own count.
      if (!RING || __ballot(min(lim0, lim1) < 27) != 0) {
        if constexpr (RING) asm volatile("");  // a branch, not 64 selections in every tile
#pragma unroll
        for (int rr = 0; rr < 16; ++rr) {
          const int off = 8 * (rr >> 2) + (rr & 3);
          s0[rr] = off > lim0 ? 0.f : s0[rr];
          s1[rr] = off > lim1 ? 0.f : s1[rr];
        }
      }
      a0 += s0;
      a1 += s1;
    };
    // The place of row r, of the last row if there is no such row.
    auto place_of = [&](int r) TASFT_INLINE {
      RowPlace at;
      at.i = r / p.G;
      at.g = r - at.i * p.G;
      return at;
    };
    const int64_t head0 = (int64_t)kvh * p.G;

    if constexpr (RING) {
      constexpr int STEP = OWN ? WAVES * 32 : kTile;   // rows of a step
      constexpr int SHARE = OWN ? 32 : STEP / WAVES;   // of them, a wave's share of the copying
      constexpr int UNITS = SHARE / RPU;
      constexpr int TILES = OWN ? 1 : 2;               // 32 rows that a wave adds in a step
      const int di = STEP / p.G, dg = STEP - di * p.G;
      const int r_start = r_first / STEP * STEP;
      const int steps = (rows - r_start + STEP - 1) / STEP;
      // Byte offsets of the rows a lane brings, moved a step at a time (the host sees to it that 32
      // bits hold them). The buffers end with the sequence's last row: rows past it are zeros.
      const int tokb = (int)p.sq[0] * 2, headb = (int)p.sq[1] * 2;
      const int tokl = (int)wp.sl[0] * 4, headl = (int)wp.sl[1] * 4;
      const __amdgpu_buffer_rsrc_t qr = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(p.q + (int64_t)sq.t0 * p.sq[0] + head0 * p.sq[1]), (short)0,
          (sq.len - 1) * tokb + (p.G - 1) * headb + ROWB, 0x00020000);
      const __amdgpu_buffer_rsrc_t lr = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(wp.lse + (int64_t)sq.t0 * wp.sl[0] + head0 * wp.sl[1]), (short)0,
          (sq.len - 1) * tokl + (p.G - 1) * headl + 4, 0x00020000);
      struct Source {
        int off, g;
      };
      auto move = [&](Source& x, int tb, int hb) TASFT_INLINE {
        x.off += di * tb + dg * hb;
        if (dg != 0) {
          x.g += dg;
          const bool wrap = x.g >= p.G;
          x.off += wrap ? tb - p.G * hb : 0;
          x.g -= wrap ? p.G : 0;
        }
      };
      Source src[UNITS], lsrc;
      RowPlace tile[TILES];
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        const int row = wave * SHARE + u * RPU + lane / (ROWB / 16);
        const RowPlace at = place_of(r_start + row);
        src[u] = {at.i * tokb + at.g * headb + chunk_swz_k<D>(row, lane % (ROWB / 16)) * 16, at.g};
      }
      {
        const RowPlace at = place_of(r_start + (OWN ? wave * SHARE + col : lane));
        lsrc = {at.i * tokl + at.g * headl, at.g};
      }
#pragma unroll
      for (int t = 0; t < TILES; ++t) tile[t] = place_of(r_start + (OWN ? wave * SHARE : t * 32) + col);
      auto dma_step = [&](uint8_t* stage, float* lstage) TASFT_INLINE {
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
          chunk_dma(qr, stage + (wave * SHARE + u * RPU) * ROWB, src[u].off);
          move(src[u], tokb, headb);
        }
        chunk_dma4(lr, lstage, lsrc.off);
        move(lsrc, tokl, headl);
      };
      // Adds the rows r .. r + 31 of a stage.
      auto add_tile = [&](const uint8_t* now, const float* lnow, int r, RowPlace& at, auto between) TASFT_INLINE {
        u32x4_t qf[KSTEPS];
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ++ks)
          qf[ks] = *(const u32x4_t*)(now + (r + col) * ROWB + chunk_swz_k<D>(r + col, ks * 2 + half) * 16);
        add_rows(qf, at, at.i < sq.len, lnow[OWN ? lane : r + col], between);
        at.move(di, dg, p.G);
      };
      if constexpr (OWN) {
        // The stage is filled again, for two steps on, once its rows have been used.
        auto step = [&](uint8_t* now, float* lnow) TASFT_INLINE {
          __builtin_amdgcn_s_waitcnt(vm_wait(UNITS + 1));
          add_tile(now, lnow, wave * SHARE, tile[0], [] {});
          __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
          dma_step(now, lnow);
        };
        dma_step(s0_lds, lse_lds[0][wave]);
        dma_step(s1_lds, lse_lds[1][wave]);
        for (int s = 0; s < steps; s += 2) {
          step(s0_lds, lse_lds[0][wave]);
          if (s + 1 >= steps) break;
          step(s1_lds, lse_lds[1][wave]);
        }
      } else {
        dma_step(s0_lds, lse_lds[0][wave]);
        dma_step(s1_lds, lse_lds[1][wave]);
        dma_step(s2_lds, lse_lds[2][wave]);
        // Every step issues the DMA of the one three steps on (past the end: zeros that no step
        // reads), so that the wait is for a fixed count. By the barrier every wave's share has
        // landed, and every wave is done with the stage that is filled next.
        auto step = [&](const uint8_t* now, const float* lnow, uint8_t* then, float* lthen) TASFT_INLINE {
          __builtin_amdgcn_s_waitcnt(vm_wait(2 * (UNITS + 1)));
          __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
          chunk_barrier();
          if constexpr (!MASKED) dma_step(then, lthen);
#pragma unroll
          for (int t = 0; t < TILES; ++t) add_tile(now, lnow, t * 32, tile[t], [] {});
          // Behind the mask bytes' loads: the wait for them would wait for it too.
          if constexpr (MASKED) dma_step(then, lthen);
        };
        for (int s = 0; s < steps; s += 4) {
          step(s0_lds, lse_lds[0][wave], s3_lds, lse_lds[3][wave]);
          if (s + 1 >= steps) break;
          step(s1_lds, lse_lds[1][wave], s0_lds, lse_lds[0][wave]);
          if (s + 2 >= steps) break;
          step(s2_lds, lse_lds[2][wave], s1_lds, lse_lds[1][wave]);
          if (s + 3 >= steps) break;
          step(s3_lds, lse_lds[3][wave], s2_lds, lse_lds[2][wave]);
        }
      }
      __builtin_amdgcn_s_waitcnt(0x0f70);  // no DMA into this workgroup's LDS outlives it
    } else {
      constexpr int STEP = 32 * RW;
      u32x4_t qf[KSTEPS];
      RowPlace at;
      float lse;
      auto load_rows = [&](int r0) TASFT_INLINE {  // past the end: the last row again, not used
        at = place_of(min(r0 + col, rows - 1));
        const int64_t tok = sq.t0 + at.i, h = head0 + at.g;
        const uint16_t* qr = p.q + tok * p.sq[0] + h * p.sq[1] + half * 8;
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ++ks) qf[ks] = *(const u32x4_t*)(qr + ks * 16);
        lse = wp.lse[tok * wp.sl[0] + h * wp.sl[1]];
      };
      int r0 = (r_first / 32 + rg) * 32;
      if (r0 < rows) {
        load_rows(r0);
        for (; r0 < rows; r0 += STEP)
          add_rows(qf, at, r0 + col < rows, lse, [&]() TASFT_INLINE { load_rows(r0 + STEP); });
      }
    }
    // Sums over the 32 rows of a half's lanes, halving the registers each time: lanes whose bit is
    // set go on with the upper registers' sums. Lane col ends with the sum of register col.
    float v[32];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const auto sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(a0[j]), __float_as_uint(a1[j]), false, false);
      v[j] = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    }
    auto halve = [&](auto ctrl, int n2, int bit) TASFT_INLINE {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n2) {
          const bool up = (lane & bit) != 0;
          const float mine = up ? v[j + n2] : v[j], other = up ? v[j] : v[j + n2];
          v[j] = mine + dpp_f32<decltype(ctrl)::value>(other);
        }
    };
    halve(std::integral_constant<int, 0x140>{}, 8, 8);  // row_mirror
    halve(std::integral_constant<int, 0x141>{}, 4, 4);  // row_half_mirror
    halve(std::integral_constant<int, 0x1B>{}, 2, 2);   // quad_perm [3, 2, 1, 0]
    halve(std::integral_constant<int, 0xB1>{}, 1, 1);   // quad_perm [1, 0, 3, 2]
    total = v[0];
    if constexpr (RW > 1) {
      lse_lds[0][wave][lane] = total;
      __syncthreads();
      total = (lse_lds[0][0][lane] + lse_lds[0][1][lane]) + (lse_lds[0][2][lane] + lse_lds[0][3][lane]);
      if constexpr (WAVES == 8)
        total += (lse_lds[0][4][lane] + lse_lds[0][5][lane]) + (lse_lds[0][6][lane] + lse_lds[0][7][lane]);
    }
  }
  const int key = key0 + (col >> 4) * 32 + ((col & 15) >> 2) * 8 + (col & 3) + 4 * half;
  if (rg == 0 && key < p.cap) {
    const float before = wp.scores ? wp.scores[n * wp.ss[0] + kvh * wp.ss[1] + key * wp.ss[2]] : 0.f;
    wp.out[((int64_t)n * p.Hkv + kvh) * p.cap + key] = key < sq.kv ? before + total : before;
  }
}

}  // namespace tasft

using namespace tasft;

// Whether a launch of `groups` times `each` workgroups holds fewer than 2^32 threads, as it must.
static bool launch_fits(int64_t groups, int64_t each, int threads) {
  const int64_t most = (int64_t)0xffffffff / threads;
  return groups <= most && each <= most && groups * each <= most;
}

// Checks shared by both entry points; fills the parameters that they share.
static int chunk_params(ChunkParams& p, const char* what, const void* q, const void* k_pages, const uint8_t* mask,
                        const int32_t* table, const int32_t* kv_lens, const int32_t* cu, int64_t num_seqs,
                        int64_t tokens, int64_t num_q_heads, int64_t num_kv_heads, int64_t max_seqlen,
                        int64_t head_dim, int64_t block_size, int64_t mask_rows, int64_t page_size,
                        int64_t num_pages, int64_t max_pages, const int64_t* q_strides, const int64_t* kp_strides,
                        const int64_t* mask_strides, int64_t bt_stride, float scale, int causal, int dtype) {
  if (!q || !k_pages || !table || !kv_lens || !cu || !q_strides || !kp_strides || (mask && !mask_strides))
    return set_error(kErrInvalidArgument, "%s: null pointer argument", what);
  if (dtype != kBf16 && dtype != kF16)
    return set_error(kErrUnsupported, "%s: dtype must be bf16 (0) or fp16 (1), got %d", what, dtype);
  if (num_seqs <= 0 || tokens <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || max_seqlen <= 0 || num_pages <= 0 ||
      max_pages <= 0 || (mask && mask_rows <= 0))
    return set_error(kErrInvalidArgument, "%s: sizes must be positive", what);
  if (num_q_heads % num_kv_heads != 0)
    return set_error(kErrInvalidArgument, "%s: num_q_heads must be a multiple of num_kv_heads", what);
  if (head_dim != 64 && head_dim != 128)
    return set_error(kErrUnsupported, "%s: head_dim must be 64 or 128, got %lld", what, (long long)head_dim);
  if (mask && block_size != 32 && block_size != 64 && block_size != 128)
    return set_error(kErrUnsupported, "%s: block_size must be 32, 64 or 128, got %lld", what, (long long)block_size);
  if (page_size < 8 || (page_size & (page_size - 1)))
    return set_error(kErrUnsupported, "%s: page_size must be a power of two >= 8, got %lld", what,
                     (long long)page_size);
  if (!(scale > 0.f)) return set_error(kErrInvalidArgument, "%s: scale must be positive", what);
  const int64_t lim = 0x7fffffff;
  if (num_seqs > lim - 1 || tokens > lim || num_pages > lim || page_size > lim || max_pages > lim ||
      max_pages * page_size > lim - 255 || tokens * (num_q_heads / num_kv_heads) > lim - 255 || mask_rows > lim ||
      num_q_heads > 65535)
    return set_error(kErrUnsupported, "%s: sizes exceed 32 bits", what);
  if (!strides_nonneg(q_strides, 3) || !strides_nonneg(kp_strides, 4) || bt_stride < 0 ||
      (mask && !strides_nonneg(mask_strides, 4)))
    return set_error(kErrInvalidArgument, "%s: strides must be non-negative", what);
  if (q_strides[2] != 1 || kp_strides[3] != 1)
    return set_error(kErrInvalidArgument, "%s: head dims must be contiguous", what);
  if ((q_strides[0] & 7) || (q_strides[1] & 7) || (kp_strides[0] & 7) || (kp_strides[1] & 7) ||
      (kp_strides[2] & 7) || ((uintptr_t)q & 15) || ((uintptr_t)k_pages & 15))
    return set_error(kErrInvalidArgument, "%s: strides must be multiples of 8 on 16-byte aligned bases", what);
  if (kp_strides[1] >= (int64_t)1 << 24)
    return set_error(kErrUnsupported, "%s: token stride of the pools too large", what);
  p.q = (const uint16_t*)q;
  p.k = (const uint16_t*)k_pages;
  p.mask = mask;
  p.table = table;
  p.kv_lens = kv_lens;
  p.cu = cu;
  p.sq[0] = q_strides[0];
  p.sq[1] = q_strides[1];
  for (int i = 0; i < 3; ++i) p.sk[i] = kp_strides[i];
  if (mask)
    for (int i = 0; i < 4; ++i) p.sm[i] = mask_strides[i];
  p.bt_stride = bt_stride;
  p.N = (int)num_seqs;
  p.T = (int)tokens;
  p.Hq = (int)num_q_heads;
  p.Hkv = (int)num_kv_heads;
  p.G = (int)(num_q_heads / num_kv_heads);
  p.L = (int)(max_seqlen < tokens ? max_seqlen : tokens);
  p.ps_shift = __builtin_ctzll((unsigned long long)page_size);
  p.num_pages = (int)num_pages;
  p.cap = (int)(max_pages * page_size);
  p.bs_shift = mask ? __builtin_ctzll((unsigned long long)block_size) : 6;
  p.mask_rows = (int)mask_rows;
  p.scale_log2 = scale * kLog2e;
  p.causal = causal;
  p.P = 1;
  return kOk;
}

extern "C" size_t tasft_chunk_workspace_bytes(int64_t tokens, int64_t num_q_heads, int64_t head_dim,
                                              int64_t num_splits) {
  if (tokens <= 0 || num_q_heads <= 0 || head_dim <= 0 || num_splits <= 1) return 0;
  return (size_t)(tokens * num_q_heads * num_splits) * (size_t)(head_dim + 2) * sizeof(float);
}

// Rows of a workgroup that joins few splits.
constexpr int join_rows(int64_t head_dim) { return 256 / (int)(head_dim / 4); }

template <int D, int DT>
static int launch_chunk(const ChunkParams& p, int mask, int64_t grid, hipStream_t stream) {
  auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(mask == kPositions ? 128 : 256), 0, stream, p);
  };
  if (mask == kPositions) {
    if (p.ps_shift >= 5) run(chunk_rows_kernel<D, DT, kPositions, 1>);
    else if (p.ps_shift == 4) run(chunk_rows_kernel<D, DT, kPositions, 2>);
    else run(chunk_rows_kernel<D, DT, kPositions, 4>);
  } else if (mask == kRows) {
    if (p.ps_shift >= 4) run(chunk_rows_kernel<D, DT, kRows, 1>);
    else run(chunk_rows_kernel<D, DT, kRows, 2>);
  } else {
    if (p.ps_shift >= 4) run(chunk_rows_kernel<D, DT, kDense, 1>);
    else run(chunk_rows_kernel<D, DT, kDense, 2>);
  }
  if (const int rc = check_launch("chunk attention")) return rc;
  if (p.P == 1) return kOk;
  const int64_t rows = (int64_t)p.T * p.Hq;
  if (p.P <= kFewSplits) {
    constexpr int RPW = join_rows(D);
    hipLaunchKernelGGL((chunk_combine_few_kernel<D, DT>), dim3((unsigned)((rows + RPW - 1) / RPW)), dim3(256), 0,
                       stream, p);
  } else {
    hipLaunchKernelGGL((chunk_combine_kernel<D, DT>), dim3((unsigned)rows), dim3(256), 0, stream, p);
  }
  return check_launch("chunk combine");
}

extern "C" int tasft_chunk_paged_fwd(
    const void* q, const void* k_pages, const void* v_pages, void* out, float* lse, const uint8_t* block_mask,
    const int32_t* block_table, const int32_t* kv_lens, const int32_t* cu_seqlens, void* workspace,
    size_t workspace_bytes, int64_t num_seqs, int64_t tokens, int64_t num_q_heads, int64_t num_kv_heads,
    int64_t max_seqlen, int64_t head_dim, int64_t block_size, int64_t mask_rows, int64_t page_size,
    int64_t num_pages, int64_t max_pages, int64_t num_splits, const int64_t* q_strides, const int64_t* kp_strides,
    const int64_t* vp_strides, const int64_t* o_strides, const int64_t* mask_strides, int64_t block_table_stride,
    float scale, int causal, int dtype, void* stream) {
  const char* what = "chunk attention";
  ChunkParams p = {};
  if (!v_pages || !out || !vp_strides || !o_strides)
    return set_error(kErrInvalidArgument, "chunk attention: null pointer argument");
  if (const int rc = chunk_params(p, what, q, k_pages, block_mask, block_table, kv_lens, cu_seqlens, num_seqs, tokens,
                                  num_q_heads, num_kv_heads, max_seqlen, head_dim, block_size, mask_rows, page_size,
                                  num_pages, max_pages, q_strides, kp_strides, mask_strides, block_table_stride,
                                  scale, causal, dtype))
    return rc;
  if (!strides_nonneg(vp_strides, 4) || !strides_nonneg(o_strides, 3))
    return set_error(kErrInvalidArgument, "chunk attention: strides must be non-negative");
  if (vp_strides[3] != 1 || o_strides[2] != 1)
    return set_error(kErrInvalidArgument, "chunk attention: head dims must be contiguous");
  if ((vp_strides[0] & 7) || (vp_strides[1] & 7) || (vp_strides[2] & 7) || (o_strides[0] & 7) || (o_strides[1] & 7) ||
      ((uintptr_t)v_pages & 15) || ((uintptr_t)out & 15))
    return set_error(kErrInvalidArgument, "chunk attention: strides must be multiples of 8 on 16-byte aligned bases");
  if (vp_strides[1] >= (int64_t)1 << 24)
    return set_error(kErrUnsupported, "chunk attention: token stride of the pools too large");
  if (num_splits < 1 || num_splits > 1024)
    return set_error(kErrInvalidArgument, "chunk attention: num_splits must be in [1, 1024]");
  if (num_splits > 1 &&
      (!workspace || workspace_bytes < tasft_chunk_workspace_bytes(tokens, num_q_heads, head_dim, num_splits)))
    return set_error(kErrWorkspace, "chunk attention: workspace too small");
  if ((uintptr_t)workspace & 15)
    return set_error(kErrInvalidArgument, "chunk attention: workspace must be 16-byte aligned");
  p.v = (const uint16_t*)v_pages;
  p.o = (uint16_t*)out;
  p.lse = lse;
  for (int i = 0; i < 3; ++i) p.sv[i] = vp_strides[i];
  p.so[0] = o_strides[0];
  p.so[1] = o_strides[1];
  p.P = (int)num_splits;
  p.ws_o = (float*)workspace;
  p.ws_ml = (float*)workspace + tokens * num_q_heads * num_splits * head_dim;
  // Row tiles: masked ones are aligned to positions, so a chunk can touch one more.
  // Up to a wave's rows the heads of a group share K and V: 61 sequences of 1099 keys, 4 heads a KV head,
  // a fourth of the blocks of 32, 26 us and as positions of each head 44; 32 sequences of 4096, 32 heads
  // a KV head, 28 and 93; a tenth of the blocks of 64 sequences of 16384, 4 heads, 297 both ways, of 8
  // sequences of 8192 33 and 30.
  const int form = !p.mask ? kDense : (int64_t)p.L * p.G <= 32 ? kRows : kPositions;
  const int64_t rows = form == kPositions ? (int64_t)p.L + kMaskTile - 1 : (int64_t)p.L * p.G;
  const int tile = form == kPositions ? kMaskTile : kRowTile;
  p.QT = (int)((rows + tile - 1) / tile);
  const int64_t groups = (int64_t)p.N * p.Hkv, each = (int64_t)p.QT * (form == kPositions ? p.G : 1) * p.P;
  const int64_t out_rows = (int64_t)p.T * p.Hq, joined = p.P <= kFewSplits ? join_rows(head_dim) : 1;
  if (!launch_fits(groups, each, form == kPositions ? 128 : 256) ||
      (p.P > 1 && !launch_fits((out_rows + joined - 1) / joined, 1, 256)))
    return set_error(kErrUnsupported, "chunk attention: launch too large");
  const int64_t grid = groups * each;
  const hipStream_t st = (hipStream_t)stream;
  if (head_dim == 128)
    return dtype == kF16 ? launch_chunk<128, kF16>(p, form, grid, st) : launch_chunk<128, kBf16>(p, form, grid, st);
  return dtype == kF16 ? launch_chunk<64, kF16>(p, form, grid, st) : launch_chunk<64, kBf16>(p, form, grid, st);
}

template <int D, int DT>
static void launch_weights(const WeightParams& w, hipStream_t stream) {
  const ChunkParams& p = w.c;
  const int64_t heads = (int64_t)p.N * p.Hkv;
  auto grid = [&](int kw) { return heads * ((p.cap + kw * kTile - 1) / (kw * kTile)); };
  // Byte offsets within a sequence's rows of Q and log-sums, the steps past the end included.
  const int64_t most = ((int64_t)1 << 31) - 1, past = (int64_t)p.L + 4 * 256;
  const bool small = past * p.sq[0] * 2 + p.G * p.sq[1] * 2 + D * 2 < most &&
                     past * w.sl[0] * 4 + p.G * w.sl[1] * 4 + 4 < most;
  auto run = [&](auto plain, auto masked, int kw, bool ringed) {
    const dim3 wgs((unsigned)grid(kw)), threads(weight_waves(kw, ringed) * kWave);
    if (p.mask) hipLaunchKernelGGL(masked, wgs, threads, 0, stream, w);
    else hipLaunchKernelGGL(plain, wgs, threads, 0, stream, w);
  };
  const int64_t rows = (int64_t)p.L * p.G;
  // Few keys (not two workgroups of 256 keys per CU): four times as many workgroups (8 heads, 2048
  // keys: 512 new tokens 18 instead of 57 us, 2048 new tokens 44 instead of 193; where 64 heads have
  // 4096 keys the other way round, 64 new tokens 115 instead of 35 us).
  // Many rows: through LDS. With steps of 64 rows that pays from 33 on (8 requests of 16384 keys: 32
  // rows 52 us without and 55 with it, 64 rows 69 and 58), with steps of 256 from about 1024 on (4096
  // keys: 512 rows of one request 15 and 18 us, of two 30 and 33; 1024 of one 22 and 23, of two 56 and
  // 43; 8192 of one, 2048 keys, 64 and 44).
  if (grid(4) < 512) {
    if (small && rows >= 1024)
      run(chunk_weights_kernel<D, DT, 1, true, false>, chunk_weights_kernel<D, DT, 1, true, true>, 1, true);
    else
      run(chunk_weights_kernel<D, DT, 1, false, false>, chunk_weights_kernel<D, DT, 1, false, true>, 1, false);
  } else {
    if (small && rows > 32)
      run(chunk_weights_kernel<D, DT, 4, true, false>, chunk_weights_kernel<D, DT, 4, true, true>, 4, true);
    else
      run(chunk_weights_kernel<D, DT, 4, false, false>, chunk_weights_kernel<D, DT, 4, false, true>, 4, false);
  }
}

extern "C" int tasft_key_weights(
    const void* q, const void* k_pages, const uint8_t* block_mask, const int32_t* block_table,
    const int32_t* kv_lens, const int32_t* cu_seqlens, const float* lse, const float* scores, float* scores_out,
    int64_t num_seqs, int64_t tokens, int64_t num_q_heads, int64_t num_kv_heads, int64_t max_seqlen,
    int64_t head_dim, int64_t block_size, int64_t mask_rows, int64_t page_size, int64_t num_pages,
    int64_t max_pages, const int64_t* q_strides, const int64_t* kp_strides, const int64_t* lse_strides,
    const int64_t* score_strides, const int64_t* mask_strides, int64_t block_table_stride, float scale, int causal,
    int dtype, void* stream) {
  const char* what = "key weights";
  WeightParams w = {};
  if (!lse || !scores_out || !lse_strides || (scores && !score_strides))
    return set_error(kErrInvalidArgument, "key weights: null pointer argument");
  if (const int rc = chunk_params(w.c, what, q, k_pages, block_mask, block_table, kv_lens, cu_seqlens, num_seqs,
                                  tokens, num_q_heads, num_kv_heads, max_seqlen, head_dim, block_size, mask_rows,
                                  page_size, num_pages, max_pages, q_strides, kp_strides, mask_strides,
                                  block_table_stride, scale, causal, dtype))
    return rc;
  if (!strides_nonneg(lse_strides, 2) || (scores && !strides_nonneg(score_strides, 3)))
    return set_error(kErrInvalidArgument, "key weights: strides must be non-negative");
  // At the workgroups of many keys: those of few are fewer than 2048.
  if (!launch_fits(num_seqs * num_kv_heads, ((int64_t)w.c.cap + 4 * kTile - 1) / (4 * kTile), 256))
    return set_error(kErrUnsupported, "key weights: launch too large");
  w.scores = scores;
  if (scores)
    for (int i = 0; i < 3; ++i) w.ss[i] = score_strides[i];
  w.out = scores_out;
  w.lse = lse;
  w.sl[0] = lse_strides[0];
  w.sl[1] = lse_strides[1];
  const hipStream_t st = (hipStream_t)stream;
  if (head_dim == 128)
    dtype == kF16 ? launch_weights<128, kF16>(w, st) : launch_weights<128, kBf16>(w, st);
  else
    dtype == kF16 ? launch_weights<64, kF16>(w, st) : launch_weights<64, kBf16>(w, st);
  return check_launch(what);
}
