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
// prefix over those counts places them. The second copies rows, many workgroups per head.
// Sources lie behind n', destinations before it: no row is read and written. The second is bound
// by the bytes of the moved rows (20.8 us for 32 heads of 4096 kept of up to 32768 keys of 128, 118 MB
// in and out by the counters), the first by its chain of barriers: one workgroup a head, since the
// digits follow each other (37.8 us for the same, 12.1 for 256 heads of 1040 slots).
#include "common.h"

#include "../../include/tasft_amd.h"

namespace tasft {

constexpr int kBins = 2048;
constexpr int kMoveThreads = 256;

struct EvictParams {
  const float* scores;       // [N, Hkv, cap], strides ss
  const int32_t* positions;  // [N, Hkv, cap], strides sp
  int64_t ss[3], sp[3];
  float* scores_out;         // [N, Hkv, cap] contiguous
  int32_t* positions_out;
  const int32_t* kv_lens;
  int32_t* kv_lens_out;
  int32_t* moves;  // [N * Hkv][1 + 2 * budget]: count, holes, sources
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

// THREADS threads with KPT slots each, THREADS * KPT slots at a time: a thread's slots are
// THREADS apart, so that a round of all threads is a run of slots in order. Where a head has more
// slots (MANY), the runs of slots are taken one after the other, in each of the passes.
template <int THREADS, int KPT, bool MANY>
__global__ void __launch_bounds__(THREADS) evict_select_kernel(const EvictParams p) {
  constexpr int WAVES = THREADS / kWave;
  constexpr int RUN = THREADS * KPT;
  constexpr int CELLS = WAVES * KPT;    // (round, wave) pairs of a run, in slot order
  constexpr int BPT = kBins / THREADS;  // bins a thread sums up
  static_assert(CELLS <= THREADS, "one thread a cell");
  __shared__ uint32_t hist[3][kBins];
  __shared__ int cells[3][CELLS], base[3][CELLS];
  __shared__ int wtmp[WAVES];
  __shared__ int s_newest;
  __shared__ uint32_t s_bin, s_left, s_count;
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

  // Slots behind the kept ones; with nothing to evict the rest is copied as it is.
  auto clear_rest = [&]() {
    for (int64_t i = keep + tid; i < p.cap; i += THREADS) {
      so[i] = 0.f;
      pout[i] = -1;
    }
  };
  if (len <= p.budget) {
    for (int i = tid; i < keep; i += THREADS) {
      so[i] = sc[i * ss];
      pout[i] = po[i * sp];
    }
    clear_rest();
    if (tid == 0) moves[0] = 0;
    return;
  }

  // Weights and positions of the first run, all loads in flight together. Up to 16 slots a thread
  // they stay in registers, beyond that (HOLD false) only until the images are formed.
  constexpr bool HOLD = KPT <= 16 && !MANY;
  const int runs = MANY ? (len + RUN - 1) / RUN : 1;
  float w[MANY ? 1 : KPT];
  int32_t pos[MANY ? 1 : KPT];
  uint32_t img[KPT];
  int newest = -0x7fffffff - 1;
#pragma unroll
  for (int r = 0; r < KPT; ++r) {
    const int i = min(r * THREADS + tid, len - 1);
    const int32_t x = po[i * sp];
    if constexpr (!MANY) {
      w[r] = sc[i * ss];
      pos[r] = x;
    }
    newest = max(newest, x);
  }
  for (int i = tid; i < 3 * kBins; i += THREADS) (&hist[0][0])[i] = 0;
  if (tid == 0) s_newest = -0x7fffffff - 1;
  __syncthreads();
  if constexpr (MANY)
    for (int i = RUN + tid; i < len; i += THREADS) newest = max(newest, po[i * sp]);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) newest = max(newest, __shfl_xor(newest, off, kWave));
  if (lane == 0) atomicMax(&s_newest, newest);
  __syncthreads();
  const int64_t first_recent = (int64_t)s_newest - p.recent;  // positions above it are recent
  auto image = [&](float weight, int32_t position) {
    return position < p.sinks || position > first_recent ? 0xffffffffu : weight_image(weight);
  };
  // The thread's number again, opaque: addresses of one pass are not kept in registers for another.
  auto again = [&]() {
    int t = tid;
    if constexpr (!HOLD) asm volatile("" : "+v"(t));
    return t;
  };
  auto form_images = [&](int run) {  // 0 for slots past the last
#pragma unroll
    for (int r0 = 0; r0 < KPT; r0 += 8) {
      const int t = again();
#pragma unroll
      for (int r = r0; r < r0 + 8; ++r) {
        const int i = run * RUN + r * THREADS + t, j = min(i, len - 1);
        const uint32_t x = MANY ? image(sc[j * ss], po[j * sp]) : image(w[MANY ? 0 : r], pos[MANY ? 0 : r]);
        img[r] = i < len ? x : 0u;
      }
      if constexpr (MANY) asm volatile("" ::: "memory");  // eight slots' loads at a time: registers
    }
  };
  form_images(0);
  auto take_run = [&](int run) {
    if constexpr (MANY) form_images(run);
  };

  // The keep-th largest image, digit by digit.
  uint32_t prefix = 0, left = (uint32_t)keep, equal = 0;
#pragma unroll
  for (int d = 0; d < 3; ++d) {
    const int shift = d == 0 ? 21 : (d == 1 ? 10 : 0);
    const int bits = d == 2 ? 10 : 11;
    const uint32_t above = d == 0 ? 0u : (0xffffffffu << (shift + bits));
    for (int run = 0; run < runs; ++run) {
      take_run(run);
#pragma unroll
      for (int r = 0; r < KPT; ++r) {
        const bool on = img[r] != 0u && (img[r] & above) == prefix;
        const uint64_t live = __ballot(on);
        if (live == 0) continue;
        // One bin for the whole wave (equal weights, protected runs): one addition.
        const uint32_t bin = (img[r] >> shift) & ((1u << bits) - 1u);
        const int lead = __builtin_ctzll(live);
        const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)bin, lead);
        if (__ballot(on && bin != first) == 0) {
          if (lane == lead) atomicAdd(&hist[d][first], (uint32_t)__popcll(live));
        } else if (on) {
          atomicAdd(&hist[d][bin], 1u);
        }
      }
    }
    __syncthreads();
    // Bins from the top: thread t sums up the BPT bins from kBins - 1 - BPT t down.
    const int top = kBins - 1 - BPT * tid;
    uint32_t c[BPT], sum = 0;
#pragma unroll
    for (int j = 0; j < BPT; ++j) sum += c[j] = hist[d][top - j];
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
        if (before < left && left <= before + c[j]) {
          s_bin = top - j;
          s_left = left - before;
          s_count = c[j];
        }
        before += c[j];
      }
    }
    __syncthreads();
    prefix |= s_bin << shift;
    left = s_left;
    equal = s_count;
  }
  // Images above `prefix` stay, and the first `left` of the `equal` ones equal to it.
  const uint32_t limit = prefix;
  const bool split_equal = left < equal;

  // Numbers of flagged slots before each (round, wave) of the run: its counts in `cells[which]`
  // to `base[which]`; carry is the number before the run.
  auto number_cells = [&](int which, int carry) {
    int x = tid < CELLS ? cells[which][tid] : 0;
    const int own = x;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const int o = __shfl_up(x, off, kWave);
      if (lane >= off) x += o;
    }
    if (lane == 63) wtmp[wave] = x;
    __syncthreads();
    int before = carry + x - own;
    for (int v = 0; v < wave; ++v) before += wtmp[v];
    if (tid < CELLS) base[which][tid] = before;
    int total = carry;
#pragma unroll
    for (int v = 0; v < WAVES; ++v) total += wtmp[v];
    __syncthreads();
    return total;
  };
  const uint64_t below = (1ull << lane) - 1ull;
  int* holes = moves + 1;
  int* sources = moves + 1 + p.budget;
  int eq_seen = 0, hole_seen = 0, move_seen = 0;
  for (int run = 0; run < runs; ++run) {
    take_run(run);
    if (split_equal) {
#pragma unroll
      for (int r = 0; r < KPT; ++r) {
        const uint64_t bal = __ballot(img[r] == limit);
        if (lane == 0) cells[0][r * WAVES + wave] = __popcll(bal);
      }
      __syncthreads();
      eq_seen = number_cells(0, eq_seen);
    }
    // One bit a round: kept.
    uint32_t kept = 0;
#pragma unroll
    for (int r = 0; r < KPT; ++r) {
      const int i = run * RUN + r * THREADS + tid;
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
    hole_seen = number_cells(1, hole_seen);
    move_seen = number_cells(2, move_seen);
#pragma unroll
    for (int r = 0; r < KPT; ++r) {
      const int i = run * RUN + r * THREADS + again();
      const bool k = (kept >> r) & 1u, hole = i < keep && !k, mover = i >= keep && k;
      const uint64_t hb = __ballot(hole), mb = __ballot(mover);
      if (hole) holes[base[1][r * WAVES + wave] + __popcll(hb & below)] = i;
      if (mover) sources[base[2][r * WAVES + wave] + __popcll(mb & below)] = i;
      if (i < keep && k) {
        so[i] = HOLD ? w[HOLD ? r : 0] : sc[i * ss];
        pout[i] = HOLD ? pos[HOLD ? r : 0] : po[i * sp];
      }
    }
    if constexpr (MANY) __syncthreads();  // base is rewritten
  }
  if (tid == 0) moves[0] = hole_seen;  // as many movers as holes
  clear_rest();
  __threadfence_block();
  __syncthreads();
  for (int r = tid; r < hole_seen; r += THREADS) {
    const int to = holes[r], from = sources[r];
    so[to] = sc[from * ss];
    pout[to] = po[from * sp];
  }
}

// Rows of K and V from the movers' slots to the holes: D / 8 lanes move one key's K row and its
// V row, 16 bytes a lane each.
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictParams p) {
  const int nh = blockIdx.y, n = nh / p.Hkv, h = nh % p.Hkv;
  const int32_t* moves = p.moves + (int64_t)nh * (1 + 2 * (int64_t)p.budget);
  const int count = moves[0];
  const int per = p.D / 8, at_once = kMoveThreads / per;
  const int sub = threadIdx.x / per, c = threadIdx.x % per;
  if (sub >= at_once) return;
  const int32_t* table = p.table + n * p.bt_stride;
  for (int r = blockIdx.x * at_once + sub; r < count; r += gridDim.x * at_once) {
    const int to = moves[1 + r], from = moves[1 + p.budget + r];
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

extern "C" size_t tasft_evict_workspace_bytes(int64_t num_seqs, int64_t num_kv_heads, int64_t budget) {
  if (num_seqs <= 0 || num_kv_heads <= 0 || budget <= 0) return 0;
  return (size_t)(num_seqs * num_kv_heads) * (size_t)(1 + 2 * budget) * sizeof(int32_t);
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
  if (workspace_bytes < tasft_evict_workspace_bytes(num_seqs, num_kv_heads, budget))
    return set_error(kErrWorkspace, "evict: workspace too small");
  EvictParams p = {};
  p.scores = scores;
  p.positions = positions;
  p.scores_out = scores_out;
  p.positions_out = positions_out;
  p.kv_lens = kv_lens;
  p.kv_lens_out = kv_lens_out;
  p.moves = (int32_t*)workspace;
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
  // thread and 36.5 with 16; 16384 slots 49 with 16 and 58 with 32; 32768 slots 94 and, run by run, 143).
  auto select = [&](auto kernel, int threads) { hipLaunchKernelGGL(kernel, dim3(heads), dim3(threads), 0, st, p); };
  if (cap <= 2048)
    select(evict_select_kernel<256, 8, false>, 256);
  else if (cap <= 8192)
    select(evict_select_kernel<1024, 8, false>, 1024);
  else if (cap <= 16384)
    select(evict_select_kernel<1024, 16, false>, 1024);
  else if (cap <= 32768)
    select(evict_select_kernel<1024, 32, false>, 1024);
  else
    select(evict_select_kernel<1024, 32, true>, 1024);
  if (const int rc = check_launch("evict select")) return rc;
  // About 16 workgroups per CU over all heads, no more than a head's rows can use: each row is a
  // chain of a table entry and two loads, so many have to be on their way.
  const int64_t rows = kMoveThreads / (head_dim / 8);
  const int64_t most = budget < cap - budget ? budget : cap - budget;  // movers of a head at the most
  if (most <= 0) return kOk;
  const int64_t want = (4096 + heads - 1) / heads, need = (most + rows - 1) / rows;
  hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)(need < want ? need : want), heads), dim3(kMoveThreads), 0, st,
                     p);
  return check_launch("evict move");
}
