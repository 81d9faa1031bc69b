// Eviction from a paged cache by accumulated attention weight.
//
// Per (sequence, KV head): of the first kv_len slots n' = min(kv_len, budget) stay, those whose
// position is among the first `sinks` or within `recent` of the newest, then those of the
// largest weight (ties to the lowest slot). The order of keys does not matter to the attention
// that reads them later, so nothing is shifted: the kept slots behind n' move into the holes
// before it, both in ascending order. That moves each such key once and no other.
//
// Two launches. The first, one workgroup per (sequence, head), finds the weight of the n'-th key
// by a radix selection (three digits of 11, 11 and 10 bits over an order-preserving image of the
// weight, bins in LDS) and numbers holes and movers: ballots count them per round and wave, one
// prefix over those counts places them. The second copies rows, many workgroups per head. Heads of
// more than 32768 slots are selected from in parts, in six launches.
// Sources lie behind n', destinations before it: no row is read and written. The second is bound
// by the bytes of the moved rows (22.8 us for 32 heads of 4096 kept of up to 32768 keys of 128, 118 MB
// in and out by the counters), the first by its chain of barriers: one workgroup a head, since the
// digits follow each other (31.8 us for the same, 12.2 for 512 heads of 1040 slots).
#include "common.h"

#include "../../include/tasft_amd.h"

namespace tasft {

constexpr int kBins = 2048;
constexpr int kMoveThreads = 256;
constexpr int64_t kMaxSlotsHeld = 32768;  // of a head, in one workgroup

struct EvictParams {
  const float* scores;       // [N, Hkv, cap], strides ss
  const int32_t* positions;  // [N, Hkv, cap], strides sp
  int64_t ss[3], sp[3];
  float* scores_out;         // [N, Hkv, cap] contiguous
  int32_t* positions_out;
  const int32_t* kv_lens;
  int32_t* kv_lens_out;
  int32_t* moves;  // [N * Hkv][1 + 2 * budget]: count, holes, sources
  int32_t* part;   // [N * Hkv][part_words(parts)]: what the parts of a head tell each other
  int parts, part_slots;  // parts a head's slots are cut into, 1: one workgroup a head
  uint16_t* k;
  uint16_t* v;
  int64_t sk[3], sv[3];  // (page, token, head)
  const int32_t* table;
  int64_t bt_stride;
  int64_t cap;
  int N, Hkv, D, budget, recent, sinks, ps_shift, num_pages;
};

// Order-preserving image of a weight: larger means heavier; NaN counts as the heaviest weight,
// -0 as 0. Never 0 or all ones.
__device__ __forceinline__ uint32_t weight_image(float w) {
  uint32_t u = __float_as_uint(w);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xfffffffeu;
  if (u == 0x80000000u) u = 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// The image that orders a head's slots: protected positions before all weights.
__device__ __forceinline__ uint32_t slot_image(const EvictParams& p, float weight, int32_t position,
                                               int64_t first_recent) {
  return position < p.sinks || position > first_recent ? 0xffffffffu : weight_image(weight);
}

// One more in `bin` for every lane that is on. One bin for the whole wave (equal weights, protected
// runs): one addition.
__device__ __forceinline__ void count_bin(uint32_t* hist, bool on, uint32_t bin) {
  const uint64_t live = __ballot(on);
  if (live == 0) return;
  const int lead = __builtin_ctzll(live);
  const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)bin, lead);
  if (__ballot(on && bin != first) == 0) {
    if ((int)(threadIdx.x & 63) == lead) atomicAdd(&hist[first], (uint32_t)__popcll(live));
  } else if (on) {
    atomicAdd(&hist[bin], 1u);
  }
}

// The bin that holds the left-th count from the top, what is left within it, its own count. Thread t
// has the counts of the bins from kBins - 1 - kBins / THREADS t down.
struct Pick {
  uint32_t bin, left, count;
};
template <int THREADS>
__device__ __forceinline__ void pick_bin(const uint32_t (&c)[kBins / THREADS], uint32_t left, int* wtmp, Pick* found) {
  constexpr int BPT = kBins / THREADS;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t sum = 0;
#pragma unroll
  for (int j = 0; j < BPT; ++j) sum += c[j];
  uint32_t incl = sum;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const uint32_t o = __shfl_up(incl, off, kWave);
    if (lane >= off) incl += o;
  }
  if (lane == 63) wtmp[wave] = (int)incl;
  __syncthreads();
  uint32_t before = incl - sum;
  for (int v = 0; v < wave; ++v) before += (uint32_t)wtmp[v];
  if (before < left && left <= before + sum) {
#pragma unroll
    for (int j = 0; j < BPT; ++j) {
      if (before < left && left <= before + c[j]) *found = {(uint32_t)(kBins - 1 - BPT * tid - j), left - before, c[j]};
      before += c[j];
    }
  }
  __syncthreads();
}

// Numbers of flagged slots before each (round, wave), from the counts of each; returns their sum.
template <int THREADS, int CELLS>
__device__ __forceinline__ int number_cells(const int* cells, int* base, int* wtmp) {
  constexpr int WAVES = THREADS / kWave;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int own = tid < CELLS ? cells[tid] : 0;
  int x = own;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const int o = __shfl_up(x, off, kWave);
    if (lane >= off) x += o;
  }
  if (lane == 63) wtmp[wave] = x;
  __syncthreads();
  int before = x - own;
  for (int v = 0; v < wave; ++v) before += wtmp[v];
  if (tid < CELLS) base[tid] = before;
  int total = 0;
#pragma unroll
  for (int v = 0; v < WAVES; ++v) total += wtmp[v];
  __syncthreads();
  return total;
}

// Slots from .. to of a head that keeps all its len keys: as they are, 0 and -1 behind them.
__device__ __forceinline__ void copy_head(const EvictParams& p, const float* sc, const int32_t* po, float* so,
                                          int32_t* pout, int len, int64_t from, int64_t to, int tid, int threads) {
  for (int64_t i = from + tid; i < to; i += threads) {
    so[i] = i < len ? sc[i * p.ss[2]] : 0.f;
    pout[i] = i < len ? po[i * p.sp[2]] : -1;
  }
}

// THREADS threads with KPT slots each, THREADS * KPT slots at the most: a thread's slots are
// THREADS apart, so that a round of all threads is a run of slots in order.
template <int THREADS, int KPT>
__global__ void __launch_bounds__(THREADS) evict_select_kernel(const EvictParams p) {
  constexpr int WAVES = THREADS / kWave;
  constexpr int CELLS = WAVES * KPT;    // (round, wave) pairs, in slot order
  constexpr int BPT = kBins / THREADS;  // bins a thread sums up
  static_assert(CELLS <= THREADS, "one thread a cell");
  __shared__ uint32_t hist[3][kBins];
  __shared__ int cells[3][CELLS], base[3][CELLS];
  __shared__ int wtmp[WAVES];
  __shared__ int s_newest;
  __shared__ Pick found;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int nh = blockIdx.x, n = nh / p.Hkv, h = nh % p.Hkv;
  const int len = (int)min((int64_t)max(p.kv_lens[n], 0), p.cap);
  const int keep = min(len, p.budget);
  const float* sc = p.scores + n * p.ss[0] + h * p.ss[1];
  const int32_t* po = p.positions + n * p.sp[0] + h * p.sp[1];
  float* so = p.scores_out + (int64_t)nh * p.cap;
  int32_t* pout = p.positions_out + (int64_t)nh * p.cap;
  int32_t* moves = p.moves + (int64_t)nh * (1 + 2 * (int64_t)p.budget);
  const int64_t ss = p.ss[2], sp = p.sp[2];
  if (h == 0 && tid == 0) p.kv_lens_out[n] = keep;

  if (len <= p.budget) {  // nothing to evict
    copy_head(p, sc, po, so, pout, len, 0, p.cap, tid, THREADS);
    if (tid == 0) moves[0] = 0;
    return;
  }

  // Weights and positions, all loads in flight together. Up to 16 slots a thread they stay in
  // registers, beyond that (HOLD false) only until the images are formed.
  constexpr bool HOLD = KPT <= 16;
  float w[KPT];
  int32_t pos[KPT];
  uint32_t img[KPT];
  int newest = -0x7fffffff - 1;
#pragma unroll
  for (int r = 0; r < KPT; ++r) {
    const int i = min(r * THREADS + tid, len - 1);
    w[r] = sc[i * ss];
    pos[r] = po[i * sp];
    newest = max(newest, pos[r]);
  }
  for (int i = tid; i < 3 * kBins; i += THREADS) (&hist[0][0])[i] = 0;
  if (tid == 0) s_newest = -0x7fffffff - 1;
  __syncthreads();
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) newest = max(newest, __shfl_xor(newest, off, kWave));
  if (lane == 0) atomicMax(&s_newest, newest);
  __syncthreads();
  const int64_t first_recent = (int64_t)s_newest - p.recent;  // positions above it are recent
  // The thread's number again, opaque: addresses of one pass are not kept in registers for another.
  auto again = [&]() {
    int t = tid;
    if constexpr (!HOLD) asm volatile("" : "+v"(t));
    return t;
  };
#pragma unroll
  for (int r = 0; r < KPT; ++r)  // 0 for slots past the last
    img[r] = r * THREADS + again() < len ? slot_image(p, w[r], pos[r], first_recent) : 0u;

  // The keep-th largest image, digit by digit.
  uint32_t prefix = 0, left = (uint32_t)keep, equal = 0;
#pragma unroll
  for (int d = 0; d < 3; ++d) {
    const int shift = d == 0 ? 21 : (d == 1 ? 10 : 0);
    const int bits = d == 2 ? 10 : 11;
    const uint32_t above = d == 0 ? 0u : (0xffffffffu << (shift + bits));
#pragma unroll
    for (int r = 0; r < KPT; ++r)
      count_bin(hist[d], img[r] != 0u && (img[r] & above) == prefix, (img[r] >> shift) & ((1u << bits) - 1u));
    __syncthreads();
    uint32_t c[BPT];
#pragma unroll
    for (int j = 0; j < BPT; ++j) c[j] = hist[d][kBins - 1 - BPT * tid - j];
    pick_bin<THREADS>(c, left, wtmp, &found);
    prefix |= found.bin << shift;
    left = found.left;
    equal = found.count;
  }
  // Images above `prefix` stay, and the first `left` of the `equal` ones equal to it.
  const uint32_t limit = prefix;
  const bool split_equal = left < equal;

  const uint64_t below = (1ull << lane) - 1ull;
  int* holes = moves + 1;
  int* sources = moves + 1 + p.budget;
  if (split_equal) {
#pragma unroll
    for (int r = 0; r < KPT; ++r) {
      const uint64_t bal = __ballot(img[r] == limit);
      if (lane == 0) cells[0][r * WAVES + wave] = __popcll(bal);
    }
    __syncthreads();
    number_cells<THREADS, CELLS>(cells[0], base[0], wtmp);
  }
  // One bit a round: kept.
  uint32_t kept = 0;
#pragma unroll
  for (int r = 0; r < KPT; ++r) {
    const int i = r * THREADS + tid;
    bool k = img[r] > limit || (img[r] == limit && !split_equal);
    if (split_equal) {
      const bool eq = img[r] == limit;
      const uint64_t bal = __ballot(eq);
      k = k || (eq && base[0][r * WAVES + wave] + __popcll(bal & below) < (int)left);
    }
    kept |= k ? 1u << r : 0u;
    const uint64_t hb = __ballot(i < keep && !k), mb = __ballot(i >= keep && k);
    if (lane == 0) {
      cells[1][r * WAVES + wave] = __popcll(hb);
      cells[2][r * WAVES + wave] = __popcll(mb);
    }
  }
  __syncthreads();
  const int hole_count = number_cells<THREADS, CELLS>(cells[1], base[1], wtmp);
  number_cells<THREADS, CELLS>(cells[2], base[2], wtmp);
#pragma unroll
  for (int r = 0; r < KPT; ++r) {
    const int i = r * THREADS + again();
    const bool k = (kept >> r) & 1u, hole = i < keep && !k, mover = i >= keep && k;
    const uint64_t hb = __ballot(hole), mb = __ballot(mover);
    if (hole) holes[base[1][r * WAVES + wave] + __popcll(hb & below)] = i;
    if (mover) sources[base[2][r * WAVES + wave] + __popcll(mb & below)] = i;
    if (i < keep && k) {
      so[i] = HOLD ? w[HOLD ? r : 0] : sc[i * ss];
      pout[i] = HOLD ? pos[HOLD ? r : 0] : po[i * sp];
    }
  }
  if (tid == 0) moves[0] = hole_count;  // as many movers as holes
}

// The same selection where a head has more slots than one workgroup holds: its slots are cut into
// parts, a workgroup each, and every step that needs all of them is a launch. PHASE 0: a part's newest
// position. 1, 2, 3: its counts of a digit of the images. 4: the kept slots are known; those below
// the budget get their values, and the part's holes and movers are counted. 5: they are numbered.
// What a phase learns from all parts (the newest position, a digit) each workgroup of the next
// sums up for itself from what the parts wrote, in their order.
constexpr int kPartThreads = 1024, kPartRounds = 8, kPartRun = kPartThreads * kPartRounds;
constexpr int kMaxParts = 64;
// Words of a head: newest, holes and movers per part; three digits (prefix, left, equal); counts.
__host__ __device__ constexpr int64_t part_words(int parts) { return 3 * parts + 9 + (int64_t)3 * parts * kBins; }

template <int PHASE>
__global__ void __launch_bounds__(kPartThreads) evict_part_kernel(const EvictParams p) {
  constexpr int WAVES = kPartThreads / kWave, CELLS = WAVES * kPartRounds, BPT = kBins / kPartThreads;
  __shared__ uint32_t hist[kBins];
  __shared__ int cells[3][CELLS], base[3][CELLS];
  __shared__ int wtmp[WAVES];
  __shared__ int s_sum[3];
  __shared__ Pick found;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int part = blockIdx.x, nh = blockIdx.y, n = nh / p.Hkv, h = nh % p.Hkv;
  const int len = (int)min((int64_t)max(p.kv_lens[n], 0), p.cap);
  const int keep = min(len, p.budget);
  const float* sc = p.scores + n * p.ss[0] + h * p.ss[1];
  const int32_t* po = p.positions + n * p.sp[0] + h * p.sp[1];
  const int64_t ss = p.ss[2], sp = p.sp[2];
  float* so = p.scores_out + (int64_t)nh * p.cap;
  int32_t* pout = p.positions_out + (int64_t)nh * p.cap;
  int32_t* moves = p.moves + (int64_t)nh * (1 + 2 * (int64_t)p.budget);
  int32_t* newest_of = p.part + (int64_t)nh * part_words(p.parts);
  int32_t* holes_of = newest_of + p.parts;
  int32_t* movers_of = holes_of + p.parts;
  uint32_t* digits = (uint32_t*)(movers_of + p.parts);
  uint32_t* counts = digits + 9;  // [digit][part][bin]
  const int64_t from = (int64_t)part * p.part_slots, to = min(from + p.part_slots, (int64_t)len);
  const int parts = (int)(((int64_t)len + p.part_slots - 1) / p.part_slots);  // that hold keys

  if constexpr (PHASE == 4) {
    if (h == 0 && part == 0 && tid == 0) p.kv_lens_out[n] = keep;
    if (len <= p.budget) {
      copy_head(p, sc, po, so, pout, len, from, min(from + p.part_slots, p.cap), tid, kPartThreads);
      if (part == 0 && tid == 0) moves[0] = 0;
    }
  }
  if (len <= p.budget || from >= len) return;

  // Sums and maxima of all threads.
  auto sum3 = [&](int a, int b, int c) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
      a += __shfl_xor(a, off, kWave);
      b += __shfl_xor(b, off, kWave);
      c += __shfl_xor(c, off, kWave);
    }
    if (tid < 3) s_sum[tid] = 0;
    __syncthreads();
    if (lane == 0) {
      atomicAdd(&s_sum[0], a);
      atomicAdd(&s_sum[1], b);
      atomicAdd(&s_sum[2], c);
    }
    __syncthreads();
  };
  auto newest_all = [&](int x) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) x = max(x, __shfl_xor(x, off, kWave));
    if (tid == 0) s_sum[0] = -0x7fffffff - 1;
    __syncthreads();
    if (lane == 0) atomicMax(&s_sum[0], x);
    __syncthreads();
    x = s_sum[0];
    __syncthreads();
    return x;
  };
  if constexpr (PHASE == 0) {
    int x = -0x7fffffff - 1;
    for (int64_t i = from + tid; i < to; i += kPartThreads) x = max(x, po[i * sp]);
    x = newest_all(x);
    if (tid == 0) newest_of[part] = x;
    return;
  } else {
    const int64_t first_recent = (int64_t)newest_all(tid < parts ? newest_of[tid] : -0x7fffffff - 1) - p.recent;
    auto image_at = [&](int64_t i) {  // 0 for slots past the part's last
      const int64_t j = min(i, to - 1);
      const uint32_t x = slot_image(p, sc[j * ss], po[j * sp], first_recent);
      return i < to ? x : 0u;
    };
    // The digits so far: PHASE - 1 of them, the last one summed up here.
    constexpr int DONE = PHASE < 4 ? PHASE - 1 : 3;
    uint32_t prefix = 0, left = (uint32_t)keep, equal = 0;
    if constexpr (PHASE == 5) {
      prefix = digits[6], left = digits[7], equal = digits[8];
    } else if constexpr (DONE > 0) {
      constexpr int d = DONE - 1, shift = d == 0 ? 21 : (d == 1 ? 10 : 0);
      if constexpr (d > 0) prefix = digits[3 * d - 3], left = digits[3 * d - 2];
      uint32_t c[BPT] = {};
      const uint32_t* of_part = counts + (int64_t)d * p.parts * kBins + kBins - 1 - BPT * tid;
      for (int q0 = 0; q0 < parts; q0 += 8) {
        uint32_t x[8][BPT];
#pragma unroll
        for (int q = 0; q < 8; ++q)
#pragma unroll
          for (int j = 0; j < BPT; ++j) x[q][j] = of_part[min(q0 + q, parts - 1) * kBins - j];
#pragma unroll
        for (int q = 0; q < 8; ++q)
#pragma unroll
          for (int j = 0; j < BPT; ++j) c[j] += q0 + q < parts ? x[q][j] : 0u;
      }
      pick_bin<kPartThreads>(c, left, wtmp, &found);
      prefix |= found.bin << shift;
      left = found.left;
      equal = found.count;
      if (part == 0 && tid == 0) {
        digits[3 * d] = prefix;
        digits[3 * d + 1] = left;
        digits[3 * d + 2] = equal;
      }
    }
    if constexpr (PHASE < 4) {
      constexpr int d = PHASE - 1, shift = d == 0 ? 21 : (d == 1 ? 10 : 0), bits = d == 2 ? 10 : 11;
      const uint32_t above = d == 0 ? 0u : (0xffffffffu << ((shift + bits) & 31));
      for (int i = tid; i < kBins; i += kPartThreads) hist[i] = 0;
      __syncthreads();
      for (int64_t i0 = from; i0 < to; i0 += kPartRun) {
        uint32_t img[kPartRounds];
#pragma unroll
        for (int r = 0; r < kPartRounds; ++r) img[r] = image_at(i0 + r * kPartThreads + tid);
#pragma unroll
        for (int r = 0; r < kPartRounds; ++r)
          count_bin(hist, img[r] != 0u && (img[r] & above) == prefix, (img[r] >> shift) & ((1u << bits) - 1u));
      }
      __syncthreads();
      for (int i = tid; i < kBins; i += kPartThreads) counts[((int64_t)d * p.parts + part) * kBins + i] = hist[i];
    } else {
      // Kept: images above `prefix`, and the first `left` of the `equal` ones equal to it. Seen in
      // the parts before this one: such equal ones, holes and movers.
      const uint32_t limit = prefix;
      const bool split_equal = left < equal, mine = tid < part;
      sum3(split_equal && mine ? (int)counts[((int64_t)2 * p.parts + tid) * kBins + (limit & 1023u)] : 0,
           PHASE == 5 && mine ? holes_of[tid] : 0, PHASE == 5 && mine ? movers_of[tid] : 0);
      int eq_seen = s_sum[0], hole_seen = s_sum[1], move_seen = s_sum[2];
      const uint64_t below = (1ull << lane) - 1ull;
      int holes = 0, movers = 0;  // of the wave, in its first lane
      for (int64_t i0 = from; i0 < to; i0 += kPartRun) {
        uint32_t img[kPartRounds];
#pragma unroll
        for (int r = 0; r < kPartRounds; ++r) img[r] = image_at(i0 + r * kPartThreads + tid);
        int eq_count = 0;
        if (split_equal) {
#pragma unroll
          for (int r = 0; r < kPartRounds; ++r) {
            const uint64_t bal = __ballot(img[r] == limit);
            if (lane == 0) cells[0][r * WAVES + wave] = __popcll(bal);
          }
          __syncthreads();
          eq_count = number_cells<kPartThreads, CELLS>(cells[0], base[0], wtmp);
        }
        uint64_t hb[kPartRounds], mb[kPartRounds];
#pragma unroll
        for (int r = 0; r < kPartRounds; ++r) {
          const int64_t i = i0 + r * kPartThreads + tid;
          bool k = img[r] > limit || (img[r] == limit && !split_equal);
          if (split_equal) {
            const bool eq = img[r] == limit;
            const uint64_t bal = __ballot(eq);
            k = k || (eq && eq_seen + base[0][r * WAVES + wave] + __popcll(bal & below) < (int)left);
          }
          hb[r] = __ballot(i < keep && !k);
          mb[r] = __ballot(i >= keep && k);
          if constexpr (PHASE == 4) {
            holes += __popcll(hb[r]);
            movers += __popcll(mb[r]);
            if (i < keep && k) {
              so[i] = sc[i * ss];
              pout[i] = po[i * sp];
            }
          } else if (lane == 0) {
            cells[1][r * WAVES + wave] = __popcll(hb[r]);
            cells[2][r * WAVES + wave] = __popcll(mb[r]);
          }
        }
        eq_seen += eq_count;
        __syncthreads();
        if constexpr (PHASE == 5) {
          const int hole_count = number_cells<kPartThreads, CELLS>(cells[1], base[1], wtmp);
          const int move_count = number_cells<kPartThreads, CELLS>(cells[2], base[2], wtmp);
#pragma unroll
          for (int r = 0; r < kPartRounds; ++r) {
            const int i = (int)(i0 + r * kPartThreads + tid);
            if (hb[r] >> lane & 1) moves[1 + hole_seen + base[1][r * WAVES + wave] + __popcll(hb[r] & below)] = i;
            if (mb[r] >> lane & 1)
              moves[1 + p.budget + move_seen + base[2][r * WAVES + wave] + __popcll(mb[r] & below)] = i;
          }
          hole_seen += hole_count;
          move_seen += move_count;
          __syncthreads();  // cells and their bases are written again
        }
      }
      if constexpr (PHASE == 4) {
        sum3(0, lane == 0 ? holes : 0, lane == 0 ? movers : 0);
        if (tid == 0) {
          holes_of[part] = s_sum[1];
          movers_of[part] = s_sum[2];
        }
      } else if (part == parts - 1 && tid == 0) {
        moves[0] = hole_seen;  // as many movers as holes
      }
    }
  }
}

// Rows of K and V from the movers' slots to the holes: D / 8 lanes move one key's K row and its
// V row, 16 bytes a lane each, and its weight and position. Slots behind the kept ones are cleared.
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictParams p) {
  const int nh = blockIdx.y, n = nh / p.Hkv, h = nh % p.Hkv;
  const int32_t* moves = p.moves + (int64_t)nh * (1 + 2 * (int64_t)p.budget);
  const int count = moves[0];
  const int64_t head = (int64_t)nh * p.cap;
  if (p.kv_lens[n] > p.budget)
    for (int64_t i = p.budget + (int64_t)blockIdx.x * kMoveThreads + threadIdx.x; i < p.cap;
         i += (int64_t)gridDim.x * kMoveThreads) {
      p.scores_out[head + i] = 0.f;
      p.positions_out[head + i] = -1;
    }
  const int per = p.D / 8, at_once = kMoveThreads / per;
  const int sub = threadIdx.x / per, c = threadIdx.x % per;
  if (sub >= at_once) return;
  const int32_t* table = p.table + n * p.bt_stride;
  for (int r = blockIdx.x * at_once + sub; r < count; r += gridDim.x * at_once) {
    const int to = moves[1 + r], from = moves[1 + p.budget + r];
    if (c == 0) {
      p.scores_out[head + to] = p.scores[n * p.ss[0] + h * p.ss[1] + from * p.ss[2]];
      p.positions_out[head + to] = p.positions[n * p.sp[0] + h * p.sp[1] + from * p.sp[2]];
    }
    const int pt = table[to >> p.ps_shift], pf = table[from >> p.ps_shift];
    if (pt < 0 || pt >= p.num_pages || pf < 0 || pf >= p.num_pages) continue;
    const int rt = to & ((1 << p.ps_shift) - 1), rf = from & ((1 << p.ps_shift) - 1);
    const u32x4_t kx = *(const u32x4_t*)(p.k + pf * p.sk[0] + rf * p.sk[1] + h * p.sk[2] + c * 8);
    const u32x4_t vx = *(const u32x4_t*)(p.v + pf * p.sv[0] + rf * p.sv[1] + h * p.sv[2] + c * 8);
    *(u32x4_t*)(p.k + pt * p.sk[0] + rt * p.sk[1] + h * p.sk[2] + c * 8) = kx;
    *(u32x4_t*)(p.v + pt * p.sv[0] + rt * p.sv[1] + h * p.sv[2] + c * 8) = vx;
  }
}

}  // namespace tasft

using namespace tasft;

// Parts of a head's slots and their length, whole runs.
static void evict_parts(int64_t cap, int* parts, int* slots) {
  *parts = 1;
  *slots = (int)cap;
  if (cap <= kMaxSlotsHeld) return;
  const int64_t runs = (cap + kPartRun - 1) / kPartRun, each = (runs + kMaxParts - 1) / kMaxParts;
  *parts = (int)((runs + each - 1) / each);
  *slots = (int)(each * kPartRun);
}

extern "C" size_t tasft_evict_workspace_bytes(int64_t num_seqs, int64_t num_kv_heads, int64_t slots, int64_t budget) {
  if (num_seqs <= 0 || num_kv_heads <= 0 || slots <= 0 || slots > 0x7ffff000 || budget <= 0) return 0;
  int parts, part_slots;
  evict_parts(slots, &parts, &part_slots);
  const int64_t words = 1 + 2 * (budget < slots ? budget : slots) + (parts > 1 ? part_words(parts) : 0);
  return (size_t)(num_seqs * num_kv_heads) * (size_t)words * sizeof(int32_t);
}

extern "C" int tasft_evict_paged(void* k_pages, void* v_pages, const int32_t* block_table, const int32_t* kv_lens,
                                 const float* scores, const int32_t* positions, int32_t* kv_lens_out,
                                 float* scores_out, int32_t* positions_out, void* workspace, size_t workspace_bytes,
                                 int64_t num_seqs, int64_t num_kv_heads, int64_t head_dim, int64_t page_size,
                                 int64_t num_pages, int64_t max_pages, int64_t budget, int64_t recent, int64_t sinks,
                                 const int64_t* kp_strides, const int64_t* vp_strides, const int64_t* score_strides,
                                 const int64_t* position_strides, int64_t block_table_stride, void* stream) {
  if (!k_pages || !v_pages || !block_table || !kv_lens || !scores || !positions || !kv_lens_out || !scores_out ||
      !positions_out || !workspace || !kp_strides || !vp_strides || !score_strides || !position_strides)
    return set_error(kErrInvalidArgument, "evict: null pointer argument");
  if (num_seqs <= 0 || num_kv_heads <= 0 || head_dim <= 0 || num_pages <= 0 || max_pages <= 0 || budget <= 0)
    return set_error(kErrInvalidArgument, "evict: sizes must be positive");
  if (recent < 0 || sinks < 0 || recent + sinks > budget)
    return set_error(kErrInvalidArgument, "evict: recent and sinks must be non-negative and fit the budget");
  if (page_size <= 0 || (page_size & (page_size - 1)) || page_size > (1 << 30))
    return set_error(kErrUnsupported, "evict: page_size must be a power of two, got %lld", (long long)page_size);
  if (head_dim % 8 != 0 || head_dim > 256)
    return set_error(kErrUnsupported, "evict: head_dim must be a multiple of 8, at most 256, got %lld",
                     (long long)head_dim);
  const int64_t cap = max_pages * page_size;
  if (num_seqs * num_kv_heads > 65535 || num_pages > 0x7fffffff || max_pages > 0x7fffffff || cap > 0x7ffff000 ||
      budget > 0x3fffffff)
    return set_error(kErrUnsupported, "evict: sizes exceed the kernels' range");
  if (!strides_nonneg(kp_strides, 4) || !strides_nonneg(vp_strides, 4) || !strides_nonneg(score_strides, 3) ||
      !strides_nonneg(position_strides, 3) || block_table_stride < 0)
    return set_error(kErrInvalidArgument, "evict: strides must be non-negative");
  if (kp_strides[3] != 1 || vp_strides[3] != 1)
    return set_error(kErrInvalidArgument, "evict: head dims must be contiguous");
  for (int i = 0; i < 3; ++i)
    if ((kp_strides[i] & 7) || (vp_strides[i] & 7))
      return set_error(kErrInvalidArgument, "evict: pool strides must be multiples of 8");
  if (((uintptr_t)k_pages & 15) || ((uintptr_t)v_pages & 15))
    return set_error(kErrInvalidArgument, "evict: pools must be 16-byte aligned");
  budget = budget < cap ? budget : cap;
  if (workspace_bytes < tasft_evict_workspace_bytes(num_seqs, num_kv_heads, cap, budget))
    return set_error(kErrWorkspace, "evict: workspace too small");
  // Later launches (and other workgroups) read the lengths, weights and positions again.
  if (kv_lens_out == kv_lens || scores_out == scores || positions_out == positions)
    return set_error(kErrInvalidArgument, "evict: outputs may not be the inputs");
  EvictParams p = {};
  p.scores = scores;
  p.positions = positions;
  p.scores_out = scores_out;
  p.positions_out = positions_out;
  p.kv_lens = kv_lens;
  p.kv_lens_out = kv_lens_out;
  p.moves = (int32_t*)workspace;
  evict_parts(cap, &p.parts, &p.part_slots);
  p.part = p.moves + num_seqs * num_kv_heads * (1 + 2 * budget);
  p.k = (uint16_t*)k_pages;
  p.v = (uint16_t*)v_pages;
  for (int i = 0; i < 3; ++i) {
    p.ss[i] = score_strides[i];
    p.sp[i] = position_strides[i];
    p.sk[i] = kp_strides[i];
    p.sv[i] = vp_strides[i];
  }
  p.table = block_table;
  p.bt_stride = block_table_stride;
  p.cap = cap;
  p.N = (int)num_seqs;
  p.Hkv = (int)num_kv_heads;
  p.D = (int)head_dim;
  p.budget = (int)budget;
  p.recent = (int)(recent < 0x7fffffff ? recent : 0x7fffffff);
  p.sinks = (int)(sinks < 0x7fffffff ? sinks : 0x7fffffff);
  p.ps_shift = __builtin_ctzll((unsigned long long)page_size);
  p.num_pages = (int)num_pages;
  const hipStream_t st = (hipStream_t)stream;
  const unsigned heads = (unsigned)(num_seqs * num_kv_heads);
  // The smallest form that holds a head's slots in registers (8 heads, half of the slots kept, both
  // launches: 2048 slots 15.2 us with 256 threads and 15.9 with 1024; 4 x 8192 slots 30.5 with 8 a
  // thread and 36.5 with 16; 16384 slots 49 with 16 and 58 with 32). Past 32768 slots in parts (8 heads
  // cut to 8192 keys: 32768 slots 48 and in parts 63; 40000 slots 64, one workgroup run by run 133;
  // 131072 slots 70 and 332, a million 206 and 3690).
  auto select = [&](auto kernel, int threads) { hipLaunchKernelGGL(kernel, dim3(heads), dim3(threads), 0, st, p); };
  if (cap <= 2048) {
    select(evict_select_kernel<256, 8>, 256);
  } else if (cap <= 8192) {
    select(evict_select_kernel<1024, 8>, 1024);
  } else if (cap <= 16384) {
    select(evict_select_kernel<1024, 16>, 1024);
  } else if (cap <= kMaxSlotsHeld) {
    select(evict_select_kernel<1024, 32>, 1024);
  } else {
    auto phase = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)p.parts, heads), dim3(kPartThreads), 0, st, p);
    };
    phase(evict_part_kernel<0>);
    phase(evict_part_kernel<1>);
    phase(evict_part_kernel<2>);
    phase(evict_part_kernel<3>);
    phase(evict_part_kernel<4>);
    phase(evict_part_kernel<5>);
  }
  if (const int rc = check_launch("evict select")) return rc;
  // About 16 workgroups per CU over all heads, no more than a head's rows (and the slots to clear, 16
  // a thread) can use: each row is a chain of a table entry and two loads, so many have to be on their
  // way (four times as many: 512 heads of 4096 slots 100 instead of 94 us, both launches, 32 of 32768
  // slots 48.5 and 48.7).
  const int64_t rows = kMoveThreads / (head_dim / 8);
  const int64_t most = budget < cap - budget ? budget : cap - budget;  // movers of a head at the most
  if (most <= 0) return kOk;
  const int64_t want = (4096 + heads - 1) / heads, clear = (cap - budget) / (16 * kMoveThreads);
  const int64_t need = (most + rows - 1) / rows > clear ? (most + rows - 1) / rows : clear;
  hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)(need < want ? need : want), heads), dim3(kMoveThreads), 0, st,
                     p);
  return check_launch("evict move");
}
