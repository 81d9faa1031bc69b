// Eviction from a paged cache by accumulated attention weight.
//
// Per (sequence, KV head): of the first kv_len slots n' = min(kv_len, budget) stay, those whose
// position is among the first `sinks` or within `recent` of the newest, then those of the
// largest weight (ties to the lowest slot). The order of keys does not matter to the attention
// that reads them later, so nothing is shifted: the kept slots behind n' move into the holes
// before it, both in ascending order. That moves each such key once and no other.
//
// Two launches. The first, one workgroup of 1024 threads per (sequence, head), finds the
// weight of the n'-th key by a radix selection (three digits of 11, 11 and 10 bits over an
// order-preserving image of the weight) and numbers holes and movers with ballots; a thread
// keeps the images of its slots in registers (up to 32 of them, 32768 slots; beyond that they
// are read again). The second copies rows, many workgroups per head. Sources lie behind n',
// destinations before it: no row is read and written. Bound by the bytes of the moved rows and
// of weights and positions, in small calls by the selection's chain of barriers.
#include "common.h"

#include "../../include/tasft_amd.h"

namespace tasft {

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / kWave;
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

// Exclusive prefix over the workgroup, in thread order, of a flag; `total` receives the sum.
// `tmp` holds kSelWaves ints; a barrier separates two uses of one `tmp`.
__device__ __forceinline__ int block_rank(bool f, int* tmp, int lane, int wave, int& total) {
  const uint64_t bal = __ballot(f);
  if (lane == 0) tmp[wave] = __popcll(bal);
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSelWaves; ++w) {
    const int c = tmp[w];
    before += w < wave ? c : 0;
    all += c;
  }
  total = all;
  return before + __popcll(bal & ((1ull << lane) - 1ull));
}

// KPT: images a thread keeps (0: none, they are formed again from memory).
template <int KPT>
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictParams p) {
  __shared__ uint32_t hist[kBins];
  __shared__ int wtmp[3][kSelWaves];
  __shared__ int s_newest;
  __shared__ uint32_t s_bin, s_left;
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
  for (int64_t i = keep + tid; i < p.cap; i += kSelThreads) {
    so[i] = 0.f;
    pout[i] = -1;
  }
  if (len <= p.budget) {
    for (int i = tid; i < keep; i += kSelThreads) {
      so[i] = sc[i * ss];
      pout[i] = po[i * sp];
    }
    if (tid == 0) moves[0] = 0;
    return;
  }

  if (tid == 0) s_newest = -0x7fffffff - 1;
  __syncthreads();
  int newest = -0x7fffffff - 1;
  for (int i = tid; i < len; i += kSelThreads) newest = max(newest, po[i * sp]);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) newest = max(newest, __shfl_xor(newest, off, kWave));
  if (lane == 0) atomicMax(&s_newest, newest);
  __syncthreads();
  const int64_t first_recent = (int64_t)s_newest - p.recent;  // positions above it are recent
  auto image_at = [&](int i) -> uint32_t {
    const int32_t pos = po[i * sp];
    const float w = sc[i * ss];
    return pos < p.sinks || pos > first_recent ? 0xffffffffu : weight_image(w);
  };
  const int rounds = (len + kSelThreads - 1) / kSelThreads;
  uint32_t img[KPT > 0 ? KPT : 1];
  if constexpr (KPT > 0) {
#pragma unroll
    for (int r = 0; r < KPT; ++r) {
      const int i = r * kSelThreads + tid;
      img[r] = i < len ? image_at(i) : 0u;
    }
  }
  // Calls f(slot, image, in range) for this thread's slots in ascending order; every thread of
  // the workgroup makes the same number of calls.
  auto each = [&](auto f) {
    if constexpr (KPT > 0) {
#pragma unroll
      for (int r = 0; r < KPT; ++r)
        if (r < rounds) f(r * kSelThreads + tid, img[r], r * kSelThreads + tid < len);
    } else {
      for (int r = 0; r < rounds; ++r) {
        const int i = r * kSelThreads + tid;
        f(i, i < len ? image_at(i) : 0u, i < len);
      }
    }
  };

  // The keep-th largest image, digit by digit.
  uint32_t prefix = 0, left = (uint32_t)keep;
  for (int d = 0; d < 3; ++d) {
    const int shift = d == 0 ? 21 : (d == 1 ? 10 : 0);
    const int bits = d == 2 ? 10 : 11;
    const uint32_t above = d == 0 ? 0u : (0xffffffffu << (shift + bits));
    for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    each([&](int, uint32_t x, bool in) {
      const bool on = in && (x & above) == prefix;
      const uint32_t bin = (x >> shift) & ((1u << bits) - 1u);
      // One bin for the whole wave (equal weights, protected runs): one addition.
      const uint64_t live = __ballot(on);
      if (live == 0) return;
      const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)bin, __builtin_ctzll(live));
      if (__ballot(on && bin != first) == 0) {
        if (lane == __builtin_ctzll(live)) atomicAdd(&hist[first], (uint32_t)__popcll(live));
      } else if (on) {
        atomicAdd(&hist[bin], 1u);
      }
    });
    __syncthreads();
    // Bins from the top: thread t holds bins 2047 - 2t and 2046 - 2t.
    const uint32_t c0 = hist[kBins - 1 - 2 * tid], c1 = hist[kBins - 2 - 2 * tid];
    uint32_t incl = c0 + c1;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const uint32_t o = __shfl_up(incl, off, kWave);
      if (lane >= off) incl += o;
    }
    if (lane == 63) wtmp[0][wave] = (int)incl;
    __syncthreads();
    uint32_t before = incl - c0 - c1;
    for (int w = 0; w < wave; ++w) before += (uint32_t)wtmp[0][w];
    if (before < left && left <= before + c0) {
      s_bin = kBins - 1 - 2 * tid;
      s_left = left - before;
    } else if (before + c0 < left && left <= before + c0 + c1) {
      s_bin = kBins - 2 - 2 * tid;
      s_left = left - before - c0;
    }
    __syncthreads();
    prefix |= s_bin << shift;
    left = s_left;
  }
  const uint32_t limit = prefix;  // images above it stay, and the first `left` equal to it

  int eq_base = 0, hole_base = 0, move_base = 0;
  int* holes = moves + 1;
  int* sources = moves + 1 + p.budget;
  each([&](int i, uint32_t x, bool in) {
    int total;
    const int eq = eq_base + block_rank(in && x == limit, wtmp[0], lane, wave, total);
    eq_base += total;
    const bool kept = in && (x > limit || (x == limit && eq < (int)left));
    const bool front = in && i < keep;
    const int hr = hole_base + block_rank(front && !kept, wtmp[1], lane, wave, total);
    hole_base += total;
    const int mr = move_base + block_rank(kept && !front, wtmp[2], lane, wave, total);
    move_base += total;
    if (front && kept) {
      so[i] = sc[i * ss];
      pout[i] = po[i * sp];
    } else if (front) {
      holes[hr] = i;
    } else if (kept) {
      sources[mr] = i;
    }
  });
  if (tid == 0) moves[0] = hole_base;  // as many movers as holes
  __threadfence_block();
  __syncthreads();
  for (int r = tid; r < hole_base; r += kSelThreads) {
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
  const dim3 b(kSelThreads);
  if (cap <= 2 * kSelThreads)
    hipLaunchKernelGGL(evict_select_kernel<2>, dim3(heads), b, 0, st, p);
  else if (cap <= 8 * kSelThreads)
    hipLaunchKernelGGL(evict_select_kernel<8>, dim3(heads), b, 0, st, p);
  else if (cap <= 32 * kSelThreads)
    hipLaunchKernelGGL(evict_select_kernel<32>, dim3(heads), b, 0, st, p);
  else
    hipLaunchKernelGGL(evict_select_kernel<0>, dim3(heads), b, 0, st, p);
  if (const int rc = check_launch("evict select")) return rc;
  // About 16 workgroups per CU over all heads, no more than a head's rows can use.
  const int64_t rows = kMoveThreads / (head_dim / 8);
  const int64_t most = budget < cap - budget ? budget : cap - budget;  // movers of a head at the most
  if (most <= 0) return kOk;
  const int64_t want = (4096 + heads - 1) / heads, need = (most + rows - 1) / rows;
  hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)(need < want ? need : want), heads), dim3(kMoveThreads), 0, st, p);
  return check_launch("evict move");
}
