// Trees of drafted tokens: their plan, which tokens are kept, and the kept tokens' keys and values.
//
// A sequence's new tokens t0 .. t0 + len - 1 are the nodes of a tree (or several): parents[t0 + i] is a
// node before i, or anything else for a root, which follows the cache directly.
//
// All three are bound by latency: a few kilobytes, read by a chain of dependent loads. Parents are
// brought to LDS once, so that a step up a tree costs an LDS read and not a trip to L2. 64 trees of 64 nodes, 8
// deep: 3.0 us for the plan, 4.6 to accept; 4 of 500, 20 deep: 3.1 and 5.3. Kept nodes of 64 requests, 8 heads of
// 128, moved: 8.2 us from an idle card; of one request 2.5.
#include "common.h"

#include "../../include/tasft_amd.h"

namespace tasft {

constexpr int kMaxNodes = 4096;

struct DraftSeq {
  int t0, all, len;  // all: its tokens; len: those of them that max_nodes takes
};

__device__ __forceinline__ DraftSeq draft_seq(const int32_t* cu, int n, int tokens, int most) {
  DraftSeq s;
  s.t0 = min(max(cu[n], 0), tokens);
  s.all = min(max(cu[n + 1], s.t0), tokens) - s.t0;
  s.len = min(s.all, most);
  return s;
}

__device__ __forceinline__ int draft_parent(int parent, int i) { return parent < i ? max(parent, -1) : -1; }

// Rows of nodes are shared out over blockIdx.y; an item is a node and a word of its bits.
__global__ void __launch_bounds__(256) draft_tree_kernel(const int32_t* parents, const int32_t* cu, const int32_t* kv_lens,
                                                         uint64_t* ancestors, int32_t* positions, int N, int tokens,
                                                         int most, int words) {
  __shared__ int up[kMaxNodes];
  const int n = blockIdx.x, tid = threadIdx.x;
  const DraftSeq s = draft_seq(cu, n, tokens, most);
  // Nodes behind max_nodes, and tokens behind the last sequence: nothing.
  auto clear = [&](int t) {
    positions[t] = 0;
    for (int w = 0; w < words; ++w) ancestors[(int64_t)t * words + w] = 0;
  };
  if (blockIdx.y == 0) {
    for (int i = s.len + tid; i < s.all; i += 256) clear(s.t0 + i);
    const int64_t end = min(max(cu[N], 0), tokens);
    for (int64_t t = end + (int64_t)n * 256 + tid; t < tokens; t += (int64_t)N * 256) clear((int)t);
  }
  const int64_t items = (int64_t)s.len * words;
  if ((int64_t)blockIdx.y * 256 >= items) return;
  for (int i = tid; i < s.len; i += 256) up[i] = draft_parent(parents[s.t0 + i], i);
  const int start = kv_lens[n] - s.all;
  __syncthreads();
  const int64_t item = (int64_t)blockIdx.y * 256 + tid;
  if (item >= items) return;
  const int i = (int)(item / words), w = (int)(item - (int64_t)i * words);
  uint64_t bits = 0;
  int depth = -1;
  for (int a = i; a >= 0; a = up[a], ++depth)
    if (a >> 6 == w) bits |= (uint64_t)1 << (a & 63);
  ancestors[(int64_t)(s.t0 + i) * words + w] = bits;
  if (w == 0) positions[s.t0 + i] = start + depth;
}

// The deepest node that agrees with the target all the way up (the lowest of several): a workgroup a
// sequence, a lane a node. A node's word tells, of the nodes from it up to one above it, how many they are and
// whether all fit; joined with that one's word it reaches twice as far, so that a path of 4096 nodes takes 13
// rounds (157 us, most of it the path's writing by one lane; node by node 3600, and of 512 nodes 94 instead of 25). A word that another lane has just joined reaches further
// and is as true, so a round needs no second copy.
constexpr uint32_t kNoNode = kMaxNodes;  // bits 0 to 12: the node above, 13 to 25: how many, 31: all fit

template <typename T>
__global__ void __launch_bounds__(256) draft_accept_kernel(const int32_t* parents, const T* tokens_in, const T* targets,
                                                           const T* first, const int32_t* cu, int32_t* path,
                                                           int32_t* counts, T* next, int tokens, int most) {
  __shared__ int16_t up[kMaxNodes];
  __shared__ uint32_t reach[kMaxNodes];
  __shared__ uint32_t best[4];
  const int n = blockIdx.x, tid = threadIdx.x;
  const DraftSeq s = draft_seq(cu, n, tokens, most);
  for (int i = tid; i < s.len; i += 256) {
    const int p = draft_parent(parents[s.t0 + i], i);
    up[i] = (int16_t)p;
    const bool fits = p >= 0 ? tokens_in[s.t0 + i] == targets[s.t0 + p] : !first || tokens_in[s.t0 + i] == first[n];
    reach[i] = (uint32_t)fits << 31 | 1u << 13 | (p >= 0 ? (uint32_t)p : kNoNode);
  }
  auto at = [&](int i) { return __hip_atomic_load(reach + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); };
  __syncthreads();
  int more;
  do {
    more = 0;
    for (int i = tid; i < s.len; i += 256) {
      const uint32_t own = at(i);
      if ((own & 0x1fff) == kNoNode) continue;
      const uint32_t above = at(own & 0x1fff);
      const uint32_t both = (own & above & 0x80000000u) | ((own & 0x3ffe000u) + (above & 0x3ffffffu));
      __hip_atomic_store(reach + i, both, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      more |= (both & 0x1fff) != kNoNode;
    }
  } while (__syncthreads_or(more));
  uint32_t mine = 0;  // depth + 1, then the lowest index
  for (int i = tid; i < s.len; i += 256) {
    const uint32_t own = reach[i];
    if (own >> 31) mine = max(mine, (own >> 13 & 0x1fff) << 12 | (uint32_t)(kMaxNodes - 1 - i));
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) mine = max(mine, (uint32_t)__shfl_xor((int)mine, off, 64));
  if ((tid & 63) == 0) best[tid >> 6] = mine;
  __syncthreads();
  mine = max(max(best[0], best[1]), max(best[2], best[3]));
  const int count = (int)(mine >> 12), last = kMaxNodes - 1 - (int)(mine & (kMaxNodes - 1));
  int32_t* row = path + (int64_t)n * most;
  for (int i = count + tid; i < most; i += 256) row[i] = -1;
  if (tid == 0) {
    counts[n] = count;
    next[n] = count > 0 ? targets[s.t0 + last] : first ? first[n] : (T)-1;
    for (int a = last, d = count - 1; d >= 0; a = up[a], --d) row[d] = a;
  }
}

struct CommitParams {
  uint16_t* pool[2];
  int64_t st[2][3];  // (page, token, head)
  const int32_t* table;
  const int32_t* kv_lens;
  const int32_t* cu;
  const int32_t* path;
  const int32_t* counts;
  int32_t* kv_lens_out;
  int32_t* positions;  // [N][Hkv][cap] or null
  int64_t bt_stride;
  int width, Hkv, chunks, ps_shift, num_pages, cap;
};

// A lane moves one 16-byte piece of every kept token, lowest slot first: the path rises, so a slot that is
// written has been read (four at a time: slot j + 4 and behind are read later, and none of them is written
// before).
__global__ void __launch_bounds__(256) draft_commit_kernel(const CommitParams p) {
  const int n = blockIdx.x;
  const int len = max(p.cu[n + 1] - p.cu[n], 0);
  const int start = p.kv_lens[n] - len;
  const int count = min(min(max(p.counts[n], 0), p.width), len);
  if (blockIdx.y == 0 && threadIdx.x == 0) p.kv_lens_out[n] = start + count;
  const int item = blockIdx.y * 256 + threadIdx.x;
  const int per = p.Hkv * p.chunks, moved = 2 * per;
  const int32_t* path = p.path + (int64_t)n * p.width;
  const int32_t* table = p.table + n * p.bt_stride;
  if (item < moved) {
    const int which = item >= per, piece = item - which * per, h = piece / p.chunks, c = piece - h * p.chunks;
    uint16_t* base = p.pool[which] + h * p.st[which][2] + c * 8;
    auto at = [&](int slot) -> uint16_t* {
      if (slot < 0 || slot >= p.cap) return nullptr;
      const int page = table[slot >> p.ps_shift];
      if (page < 0 || page >= p.num_pages) return nullptr;
      return base + page * p.st[which][0] + (int64_t)(slot & ((1 << p.ps_shift) - 1)) * p.st[which][1];
    };
    for (int j = 0; j < count; j += 4) {
      uint16_t* to[4];
      u32x4_t x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int node = j + e < count ? path[j + e] : -1;
        to[e] = nullptr;
        if (node > j + e && node < len) {  // (a node that is in its place stays)
          const uint16_t* from = at(start + node);
          to[e] = at(start + j + e);
          if (!from) to[e] = nullptr;
          if (to[e]) x[e] = *(const u32x4_t*)from;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (to[e]) *(u32x4_t*)to[e] = x[e];
    }
  } else if (p.positions && item < moved + p.Hkv) {
    int32_t* pos = p.positions + ((int64_t)n * p.Hkv + (item - moved)) * p.cap;
    for (int j = 0; j < count; ++j) {
      const int node = path[j], from = start + node, to = start + j;
      if (node > j && node < len && to >= 0 && from < p.cap) pos[to] = pos[from];
    }
  }
}

}  // namespace tasft

using namespace tasft;

static int draft_check(const char* what, int64_t num_seqs, int64_t tokens, int64_t max_nodes) {
  if (num_seqs <= 0 || tokens <= 0 || max_nodes <= 0)
    return set_error(kErrInvalidArgument, "%s: sizes must be positive", what);
  if (max_nodes > kMaxNodes)
    return set_error(kErrUnsupported, "%s: at most %d nodes a tree, got %lld", what, kMaxNodes, (long long)max_nodes);
  if (num_seqs > 0xffffff || tokens > 0x7fffffff) return set_error(kErrUnsupported, "%s: sizes too large", what);
  return kOk;
}

extern "C" int tasft_draft_tree(const int32_t* parents, const int32_t* cu_seqlens, const int32_t* kv_lens,
                                void* ancestors, int32_t* positions, int64_t num_seqs, int64_t tokens,
                                int64_t max_nodes, void* stream) {
  const char* what = "draft tree";
  if (!parents || !cu_seqlens || !kv_lens || !ancestors || !positions)
    return set_error(kErrInvalidArgument, "draft tree: null pointer argument");
  if (const int rc = draft_check(what, num_seqs, tokens, max_nodes)) return rc;
  if ((uintptr_t)ancestors & 7) return set_error(kErrInvalidArgument, "draft tree: ancestors must be 8-byte aligned");
  const int words = (int)((max_nodes + 63) / 64);
  const int64_t nodes = max_nodes < tokens ? max_nodes : tokens;
  const dim3 grid((unsigned)num_seqs, (unsigned)((nodes * words + 255) / 256));
  if ((int64_t)grid.x * grid.y * 256 > 0xffffffffll) return set_error(kErrUnsupported, "draft tree: launch too large");
  hipLaunchKernelGGL(draft_tree_kernel, grid, dim3(256), 0, (hipStream_t)stream, parents, cu_seqlens, kv_lens,
                     (uint64_t*)ancestors, positions, (int)num_seqs, (int)tokens, (int)max_nodes, words);
  return check_launch(what);
}

extern "C" int tasft_draft_accept(const int32_t* parents, const void* draft_tokens, const void* targets,
                                  const void* first_targets, const int32_t* cu_seqlens, int32_t* path, int32_t* counts,
                                  void* next_tokens, int64_t num_seqs, int64_t tokens, int64_t max_nodes, int wide,
                                  void* stream) {
  const char* what = "draft accept";
  if (!parents || !draft_tokens || !targets || !cu_seqlens || !path || !counts || !next_tokens)
    return set_error(kErrInvalidArgument, "draft accept: null pointer argument");
  if (const int rc = draft_check(what, num_seqs, tokens, max_nodes)) return rc;
  const dim3 grid((unsigned)num_seqs);
  if (wide)
    hipLaunchKernelGGL(draft_accept_kernel<int64_t>, grid, dim3(256), 0, (hipStream_t)stream, parents,
                       (const int64_t*)draft_tokens, (const int64_t*)targets, (const int64_t*)first_targets, cu_seqlens,
                       path, counts, (int64_t*)next_tokens, (int)tokens, (int)max_nodes);
  else
    hipLaunchKernelGGL(draft_accept_kernel<int32_t>, grid, dim3(256), 0, (hipStream_t)stream, parents,
                       (const int32_t*)draft_tokens, (const int32_t*)targets, (const int32_t*)first_targets, cu_seqlens,
                       path, counts, (int32_t*)next_tokens, (int)tokens, (int)max_nodes);
  return check_launch(what);
}

extern "C" int tasft_draft_commit_paged(void* k_pages, void* v_pages, const int32_t* block_table, const int32_t* kv_lens,
                                        const int32_t* cu_seqlens, const int32_t* path, const int32_t* counts,
                                        int32_t* kv_lens_out, int32_t* slot_positions, int64_t num_seqs,
                                        int64_t max_nodes, int64_t num_kv_heads, int64_t head_dim, int64_t page_size,
                                        int64_t num_pages, int64_t max_pages, const int64_t* kp_strides,
                                        const int64_t* vp_strides, int64_t block_table_stride, void* stream) {
  const char* what = "draft commit";
  if (!k_pages || !v_pages || !block_table || !kv_lens || !cu_seqlens || (!path && max_nodes > 0) || !counts || !kv_lens_out ||
      !kp_strides || !vp_strides)
    return set_error(kErrInvalidArgument, "draft commit: null pointer argument");
  if (num_seqs <= 0 || max_nodes < 0 || num_kv_heads <= 0 || num_pages <= 0 || max_pages <= 0)
    return set_error(kErrInvalidArgument, "draft commit: sizes must be positive");
  if (head_dim <= 0 || head_dim % 8 != 0 || head_dim > 256)
    return set_error(kErrUnsupported, "draft commit: head_dim must be a multiple of 8 up to 256, got %lld",
                     (long long)head_dim);
  if (page_size <= 0 || (page_size & (page_size - 1)))
    return set_error(kErrUnsupported, "draft commit: page_size must be a power of two, got %lld", (long long)page_size);
  const int64_t lim = 0x7fffffff;
  if (num_seqs > 0xffffff || max_nodes > lim || num_kv_heads > 65535 || num_pages > lim ||
      page_size > lim || max_pages > lim || max_pages * page_size > lim)
    return set_error(kErrUnsupported, "draft commit: sizes exceed 32 bits");
  CommitParams p = {};
  const int64_t* strides[2] = {kp_strides, vp_strides};
  void* pools[2] = {k_pages, v_pages};
  for (int i = 0; i < 2; ++i) {
    const int64_t* s = strides[i];
    if (!strides_nonneg(s, 4)) return set_error(kErrInvalidArgument, "draft commit: strides must be non-negative");
    if (s[3] != 1) return set_error(kErrInvalidArgument, "draft commit: head dims must be contiguous");
    if ((s[0] & 7) || (s[1] & 7) || (s[2] & 7) || ((uintptr_t)pools[i] & 15))
      return set_error(kErrInvalidArgument, "draft commit: strides must be multiples of 8 on 16-byte aligned bases");
    p.pool[i] = (uint16_t*)pools[i];
    for (int j = 0; j < 3; ++j) p.st[i][j] = s[j];
  }
  if (block_table_stride < 0) return set_error(kErrInvalidArgument, "draft commit: strides must be non-negative");
  if (kv_lens_out == kv_lens) return set_error(kErrInvalidArgument, "draft commit: kv_lens_out must not be kv_lens");
  p.table = block_table;
  p.kv_lens = kv_lens;
  p.cu = cu_seqlens;
  p.path = path;
  p.counts = counts;
  p.kv_lens_out = kv_lens_out;
  p.positions = slot_positions;
  p.bt_stride = block_table_stride;
  p.width = (int)max_nodes;
  p.Hkv = (int)num_kv_heads;
  p.chunks = (int)(head_dim / 8);
  p.ps_shift = __builtin_ctzll((unsigned long long)page_size);
  p.num_pages = (int)num_pages;
  p.cap = (int)(max_pages * page_size);
  const int64_t items = 2 * num_kv_heads * p.chunks + (slot_positions ? num_kv_heads : 0);
  const dim3 grid((unsigned)num_seqs, (unsigned)((items + 255) / 256));
  if ((int64_t)grid.x * grid.y * 256 > 0xffffffffll) return set_error(kErrUnsupported, "draft commit: launch too large");
  hipLaunchKernelGGL(draft_commit_kernel, grid, dim3(256), 0, (hipStream_t)stream, p);
  return check_launch(what);
}
