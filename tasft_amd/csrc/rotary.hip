// Rotary position embedding, and its fusion with the write of new keys and values into the
// pages of a cache.
//
// A pair (a, b) of a row at position p, of frequency f, becomes
//   (a cos(p f) - b sin(p f), b cos(p f) + a sin(p f)) * scale,
// computed in fp32 and rounded once; the inverse (the gradient) has the sign of the sine
// turned. The pairs are (i, i + R/2) or (2i, 2i + 1) of the first R dims, the other dims are
// copied. The angle is formed in 64 bits, in revolutions, and reduced to half a revolution
// before the fp32 sine: positions of any size keep the sine's own accuracy (p f in fp32 would
// be off by 0.03 rad at p = 10^6).
//
// Bound by memory: 4 bytes per element (32768 tokens of 32 + 8 heads of 128: 113 us one after the
// other, 5.9 TB/s, 124 as the forward or backward of a training pass; 64 tokens 3 us, the launch). A
// workgroup takes a token: it computes its sines once into LDS (shared by all heads; per head they
// would cost more than the traffic), then every thread keeps one place within a row and walks the
// heads, two 16-byte vectors of the two halves at a time. (Four tokens a workgroup, one wait for the
// sines of all: 125 us where one took 117, 9.1 and 8.6 for 2048 tokens, 5.6 and 4.0 for 64.) Measured
// at 10 KB a token; tokens of few or short heads leave threads without a row, behind the same wait for
// the sines: 16384 tokens of 8 + 2 heads of 64 take 18.3 us, 2.3 TB/s, of 128 23.1 us, 3.6 TB/s.
#include "common.h"

#include "../../include/tasft_amd.h"

namespace tasft {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryMaxHeadDim = 256;

struct RotaryParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;  // append only
  uint16_t* qo;
  uint16_t* ko;  // append: the K page pool
  uint16_t* vo;  // append: the V page pool
  // Element strides: q, k, qo and (apply) ko (b, h, s); v (-, h, s); pools (page, token, head).
  int64_t sq[3], sk[3], sv[3], sqo[3], sko[3], svo[3];
  const void* pos;  // int32 or int64; append: null = the slot
  int64_t sp[2];    // position strides (b, s)
  int pos64;
  const double* inv_freq;  // [pairs]
  int64_t tokens;          // B * S (apply), T (append)
  int64_t first;           // token of the launch's first workgroup
  int S, Hq, Hkv, D, pairs;
  float scale;
  int inverse;
  // Append.
  const int32_t* table;
  int64_t bt_stride;
  const int32_t* kv_lens;
  const int32_t* cu;
  int N, ps_shift, num_pages;
  int64_t cap;  // slots of the table
  int32_t* slot_pos;  // [N, Hkv, cap] or null
};

__device__ __forceinline__ int64_t position_at(const RotaryParams& p, int64_t i) {
  return p.pos64 ? ((const int64_t*)p.pos)[i] : (int64_t)((const int32_t*)p.pos)[i];
}

// A pair turned by (cos, sin) w, with the fused operations spelled out, and always rounded as a
// pair (a single fp16 conversion would be folded into the multiply-add, which rounds once instead
// of twice): every variant of the kernel gives the same bits.
__device__ __forceinline__ float2 turn(float a, float b, float2 w) {
  return make_float2(fmaf(-b, w.y, a * w.x), fmaf(a, w.y, b * w.x));
}

// VEC elements per vector: 8 where strides, alignment and dims allow (the host decides), else 1
// (1024 tokens as above: 6 and 12 us, 32768: 117 and 225).
// A place is one vector of each half (half layout), or one vector of whole pairs
// (interleaved; at VEC 1 the pair's two elements), or VEC plain elements behind the pairs.
template <int DT, int VEC, bool INTER, bool APPEND>
__global__ void __launch_bounds__(kRotaryThreads)
rotary_kernel(const RotaryParams p) {
  __shared__ float2 cs[kRotaryMaxHeadDim / 2];
  __shared__ int64_t t_pos;
  __shared__ int64_t t_slot;  // append: slot in the sequence's cache
  __shared__ int32_t t_seq;   // append: the token's sequence, N: padding
  __shared__ int32_t t_page;  // append: its page, -1: none
  const int tid = threadIdx.x;
  const int64_t tok = p.first + blockIdx.x;

  if constexpr (APPEND) {
    // A token's sequence: the number of ends at or before it (one load per thread and 256
    // sequences, instead of a search whose steps wait for each other).
    if (tid == 0) t_seq = 0;
    __syncthreads();
    for (int n0 = 0; n0 < p.N; n0 += kRotaryThreads) {
      const int n = n0 + tid;
      const int c = __popcll(__ballot(n < p.N && p.cu[n + 1] <= tok));
      if ((tid & 63) == 0 && c) atomicAdd(&t_seq, c);
    }
    __syncthreads();
    if (tid == 0) {
      const int seq = t_seq;
      int64_t slot = -1, pos = 0;
      int page = -1;
      if (seq < p.N) {
        const int64_t start = p.cu[seq], len = p.cu[seq + 1] - start;
        // From the length as it is given: clamped to the table, tokens past its end would land on the
        // live keys before them.
        slot = max(p.kv_lens[seq], 0) - len + (tok - start);
        // Outside the table, or a page outside the pool: rotated, but nothing is written.
        if (slot >= 0 && slot < p.cap) {
          page = p.table[(int64_t)seq * p.bt_stride + (slot >> p.ps_shift)];
          if (page < 0 || page >= p.num_pages) page = -1;
        }
        pos = p.pos ? position_at(p, tok * p.sp[1]) : slot;
      }
      t_slot = slot;
      t_page = page;
      t_pos = pos;
    }
  } else if (tid == 0) {
    const int64_t b = tok / p.S, s = tok - b * p.S;
    t_pos = position_at(p, b * p.sp[0] + s * p.sp[1]);
  }
  __syncthreads();
  if (tid < p.pairs) {
    double rev = (double)t_pos * (p.inv_freq[tid] * 0.15915494309189533577);
    rev -= rint(rev);
    float s, c;
    sincospif(2.f * (float)rev, &s, &c);
    cs[tid] = make_float2(c * p.scale, (p.inverse ? -s : s) * p.scale);
  }
  __syncthreads();

  // Places per row, and this thread's.
  const int turned = INTER && VEC > 1 ? 2 * p.pairs / VEC : p.pairs / VEC;
  const int places = turned + (p.D - 2 * p.pairs) / VEC;
  const int rows_at_once = kRotaryThreads / places;
  const int place = tid % places;
  if (tid / places >= rows_at_once) return;
  const bool turns = place < turned;
  // First element of the place's vector, and of its second one (half layout, pairs at VEC 1).
  int e0, e1 = -1, pair0 = 0;
  if (!turns) {
    e0 = 2 * p.pairs + (place - turned) * VEC;
  } else if (INTER) {
    e0 = VEC > 1 ? place * VEC : 2 * place;
    if (VEC == 1) e1 = e0 + 1;
    pair0 = VEC > 1 ? place * (VEC / 2) : place;
  } else {
    e0 = place * VEC;
    e1 = p.pairs + e0;
    pair0 = e0;
  }
  const int heads = p.Hq + (APPEND ? 2 : 1) * p.Hkv;
  const int64_t b = APPEND ? 0 : tok / p.S, s = tok - b * p.S;
  for (int h = tid / places; h < heads; h += rows_at_once) {
    const uint16_t* src;
    uint16_t* dst;
    bool copy = !turns, zero = false, skip = false;
    if constexpr (APPEND) {
      const int64_t in_page = t_slot & ((1 << p.ps_shift) - 1);
      if (h < p.Hq) {
        src = p.q + tok * p.sq[2] + h * p.sq[1];
        dst = p.qo + tok * p.sqo[2] + h * p.sqo[1];
        zero = t_seq >= p.N;
      } else {
        const bool is_v = h >= p.Hq + p.Hkv;
        const int g = h - p.Hq - (is_v ? p.Hkv : 0);
        src = is_v ? p.v + tok * p.sv[2] + g * p.sv[1] : p.k + tok * p.sk[2] + g * p.sk[1];
        const int64_t* st = is_v ? p.svo : p.sko;
        skip = t_page < 0;
        dst = (is_v ? p.vo : p.ko) + (int64_t)t_page * st[0] + in_page * st[1] + g * st[2];
        copy = copy || is_v;
        if (!is_v && place == 0 && !skip && p.slot_pos)
          p.slot_pos[((int64_t)t_seq * p.Hkv + g) * p.cap + t_slot] = (int32_t)t_pos;
      }
    } else {
      if (h < p.Hq) {
        src = p.q + b * p.sq[0] + h * p.sq[1] + s * p.sq[2];
        dst = p.qo + b * p.sqo[0] + h * p.sqo[1] + s * p.sqo[2];
      } else {
        const int g = h - p.Hq;
        src = p.k + b * p.sk[0] + g * p.sk[1] + s * p.sk[2];
        dst = p.ko + b * p.sko[0] + g * p.sko[1] + s * p.sko[2];
      }
    }
    if (!skip) {
      if constexpr (VEC == 8) {
        u32x4_t x = {0u, 0u, 0u, 0u}, y = {0u, 0u, 0u, 0u};
        if (!zero) {
          x = *(const u32x4_t*)(src + e0);
          if (e1 >= 0) y = *(const u32x4_t*)(src + e1);
          if (!copy) {
            float a[8], c[8];
            unpack16x8<DT>(x, a);
            if constexpr (INTER) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 w = cs[pair0 + i];
                const float2 r = turn(a[2 * i], a[2 * i + 1], w);
                x[i] = pack16x2<DT>(r.x, r.y);
              }
            } else {
              unpack16x8<DT>(y, c);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 w0 = cs[pair0 + 2 * i], w1 = cs[pair0 + 2 * i + 1];
                const float2 r0 = turn(a[2 * i], c[2 * i], w0), r1 = turn(a[2 * i + 1], c[2 * i + 1], w1);
                x[i] = pack16x2<DT>(r0.x, r1.x);
                y[i] = pack16x2<DT>(r0.y, r1.y);
              }
            }
          }
        }
        *(u32x4_t*)(dst + e0) = x;
        if (e1 >= 0) *(u32x4_t*)(dst + e1) = y;
      } else {
        uint16_t x = 0, y = 0;
        if (!zero) {
          x = src[e0];
          if (e1 >= 0) y = src[e1];
          if (!copy) {
            const float2 r = turn(bits16_to_f32<DT>(x), bits16_to_f32<DT>(y), cs[pair0]);
            const uint32_t w = pack16x2<DT>(r.x, r.y);
            x = (uint16_t)(w & 0xffffu);
            y = (uint16_t)(w >> 16);
          }
        }
        dst[e0] = x;
        if (e1 >= 0) dst[e1] = y;
      }
    }
  }
}

// Whether rows at `base`, `n` strides apart, hold whole 16-byte vectors.
static bool vector_rows(const void* base, const int64_t* strides, int n) {
  if ((uintptr_t)base & 15) return false;
  for (int i = 0; i < n; ++i)
    if (strides[i] & 7) return false;
  return true;
}

template <bool APPEND>
static int launch_rotary(RotaryParams& p, bool vec, int interleaved, int dtype, hipStream_t stream,
                         const char* what) {
  if (p.tokens > 0x7fffffff) return set_error(kErrUnsupported, "%s: too many tokens", what);
  // A launch holds fewer than 2^32 threads: more tokens in several.
  constexpr int64_t kMost = ((int64_t)1 << 32) / kRotaryThreads - 1;
  auto run = [&](auto kernel) {
    for (p.first = 0; p.first < p.tokens; p.first += kMost) {
      const int64_t left = p.tokens - p.first;
      hipLaunchKernelGGL(kernel, dim3((unsigned)(left < kMost ? left : kMost)), dim3(kRotaryThreads), 0, stream, p);
    }
  };
  if (dtype == kF16) {
    if (vec) interleaved ? run(rotary_kernel<kF16, 8, true, APPEND>) : run(rotary_kernel<kF16, 8, false, APPEND>);
    else interleaved ? run(rotary_kernel<kF16, 1, true, APPEND>) : run(rotary_kernel<kF16, 1, false, APPEND>);
  } else {
    if (vec) interleaved ? run(rotary_kernel<kBf16, 8, true, APPEND>) : run(rotary_kernel<kBf16, 8, false, APPEND>);
    else interleaved ? run(rotary_kernel<kBf16, 1, true, APPEND>) : run(rotary_kernel<kBf16, 1, false, APPEND>);
  }
  return check_launch(what);
}

}  // namespace tasft

using namespace tasft;

static int check_rotary(const char* what, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim,
                        int64_t rotary_dim, int dtype) {
  if (dtype != kBf16 && dtype != kF16)
    return set_error(kErrUnsupported, "%s: dtype must be bf16 (0) or fp16 (1), got %d", what, dtype);
  if (num_q_heads <= 0 || num_kv_heads < 0 || head_dim <= 0)
    return set_error(kErrInvalidArgument, "%s: sizes must be positive", what);
  if (num_q_heads > 65535 || num_kv_heads > 65535)
    return set_error(kErrUnsupported, "%s: at most 65535 heads", what);
  if (head_dim > kRotaryMaxHeadDim)
    return set_error(kErrUnsupported, "%s: head_dim at most %d, got %lld", what, kRotaryMaxHeadDim,
                     (long long)head_dim);
  if (rotary_dim <= 0 || (rotary_dim & 1) || rotary_dim > head_dim)
    return set_error(kErrInvalidArgument, "%s: rotary_dim must be even, in [2, head_dim], got %lld", what,
                     (long long)rotary_dim);
  return kOk;
}

static bool whole_vectors(int64_t head_dim, int64_t rotary_dim, int interleaved) {
  return head_dim % 8 == 0 && rotary_dim % (interleaved ? 8 : 16) == 0;
}

extern "C" int tasft_rotary(const void* q, const void* k, void* q_out, void* k_out, const void* positions,
                            int positions_64, const double* inv_freq, int64_t batch, int64_t num_q_heads,
                            int64_t num_kv_heads, int64_t seq_len, int64_t head_dim, int64_t rotary_dim,
                            const int64_t* q_strides, const int64_t* k_strides, const int64_t* qo_strides,
                            const int64_t* ko_strides, const int64_t* pos_strides, int interleaved, int inverse,
                            float scale, int dtype, void* stream) {
  const char* what = "rotary";
  if (!q || !q_out || !positions || !inv_freq || !q_strides || !qo_strides || !pos_strides ||
      (num_kv_heads > 0 && (!k || !k_out || !k_strides || !ko_strides)))
    return set_error(kErrInvalidArgument, "rotary: null pointer argument");
  if (const int rc = check_rotary(what, num_q_heads, num_kv_heads, head_dim, rotary_dim, dtype)) return rc;
  if (batch <= 0 || seq_len <= 0) return set_error(kErrInvalidArgument, "rotary: sizes must be positive");
  if (seq_len > 0x7fffffff) return set_error(kErrUnsupported, "rotary: seq_len too large");
  const bool kv = num_kv_heads > 0;
  if (!strides_nonneg(q_strides, 3) || !strides_nonneg(qo_strides, 3) || !strides_nonneg(pos_strides, 2) ||
      (kv && (!strides_nonneg(k_strides, 3) || !strides_nonneg(ko_strides, 3))))
    return set_error(kErrInvalidArgument, "rotary: strides must be non-negative");
  if (q_strides[3] != 1 || qo_strides[3] != 1 || (kv && (k_strides[3] != 1 || ko_strides[3] != 1)))
    return set_error(kErrInvalidArgument, "rotary: head dims must be contiguous");
  RotaryParams p = {};
  p.q = (const uint16_t*)q;
  p.k = (const uint16_t*)k;
  p.qo = (uint16_t*)q_out;
  p.ko = (uint16_t*)k_out;
  for (int i = 0; i < 3; ++i) {
    p.sq[i] = q_strides[i];
    p.sqo[i] = qo_strides[i];
    p.sk[i] = kv ? k_strides[i] : 0;
    p.sko[i] = kv ? ko_strides[i] : 0;
  }
  p.pos = positions;
  p.pos64 = positions_64;
  p.sp[0] = pos_strides[0];
  p.sp[1] = pos_strides[1];
  p.inv_freq = inv_freq;
  p.tokens = batch * seq_len;
  p.S = (int)seq_len;
  p.Hq = (int)num_q_heads;
  p.Hkv = (int)num_kv_heads;
  p.D = (int)head_dim;
  p.pairs = (int)(rotary_dim / 2);
  p.scale = scale;
  p.inverse = inverse;
  const bool vec = whole_vectors(head_dim, rotary_dim, interleaved) && vector_rows(q, q_strides, 3) &&
                   vector_rows(q_out, qo_strides, 3) &&
                   (!kv || (vector_rows(k, k_strides, 3) && vector_rows(k_out, ko_strides, 3)));
  return launch_rotary<false>(p, vec, interleaved, dtype, (hipStream_t)stream, what);
}

extern "C" int tasft_rotary_append_paged(
    const void* q, const void* k, const void* v, void* q_out, void* k_pages, void* v_pages,
    const int32_t* block_table, const int32_t* kv_lens, const int32_t* cu_seqlens, const void* positions,
    int positions_64, const double* inv_freq, int32_t* slot_positions, int64_t num_seqs, int64_t tokens,
    int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim, int64_t rotary_dim, int64_t page_size,
    int64_t num_pages, int64_t max_pages, const int64_t* q_strides, const int64_t* k_strides,
    const int64_t* v_strides, const int64_t* qo_strides, const int64_t* kp_strides, const int64_t* vp_strides,
    int64_t block_table_stride, int64_t pos_stride, int interleaved, float scale, int dtype, void* stream) {
  const char* what = "rotary append";
  if (!q || !k || !v || !q_out || !k_pages || !v_pages || !block_table || !kv_lens || !cu_seqlens || !inv_freq ||
      !q_strides || !k_strides || !v_strides || !qo_strides || !kp_strides || !vp_strides)
    return set_error(kErrInvalidArgument, "rotary append: null pointer argument");
  if (const int rc = check_rotary(what, num_q_heads, num_kv_heads, head_dim, rotary_dim, dtype)) return rc;
  if (num_kv_heads <= 0 || num_seqs <= 0 || tokens < 0 || num_pages <= 0 || max_pages <= 0)
    return set_error(kErrInvalidArgument, "rotary append: sizes must be positive");
  if (num_seqs > 0x7ffffffe || num_pages > 0x7fffffff || tokens > 0x7fffffff)
    return set_error(kErrUnsupported, "rotary append: sizes exceed 32 bits");
  if (page_size <= 0 || (page_size & (page_size - 1)) || page_size > (1 << 30))
    return set_error(kErrUnsupported, "rotary append: page_size must be a power of two, got %lld",
                     (long long)page_size);
  if (!strides_nonneg(q_strides, 2) || !strides_nonneg(k_strides, 2) || !strides_nonneg(v_strides, 2) ||
      !strides_nonneg(qo_strides, 2) || !strides_nonneg(kp_strides, 3) || !strides_nonneg(vp_strides, 3) ||
      block_table_stride < 0 || pos_stride < 0)
    return set_error(kErrInvalidArgument, "rotary append: strides must be non-negative");
  if (q_strides[2] != 1 || k_strides[2] != 1 || v_strides[2] != 1 || qo_strides[2] != 1 || kp_strides[3] != 1 ||
      vp_strides[3] != 1)
    return set_error(kErrInvalidArgument, "rotary append: head dims must be contiguous");
  if (tokens == 0) return kOk;
  RotaryParams p = {};
  p.q = (const uint16_t*)q;
  p.k = (const uint16_t*)k;
  p.v = (const uint16_t*)v;
  p.qo = (uint16_t*)q_out;
  p.ko = (uint16_t*)k_pages;
  p.vo = (uint16_t*)v_pages;
  // (token, head, dim) strides into the (b, h, s) slots; pools (page, token, head, dim) as they are.
  p.sq[1] = q_strides[1], p.sq[2] = q_strides[0];
  p.sk[1] = k_strides[1], p.sk[2] = k_strides[0];
  p.sv[1] = v_strides[1], p.sv[2] = v_strides[0];
  p.sqo[1] = qo_strides[1], p.sqo[2] = qo_strides[0];
  for (int i = 0; i < 3; ++i) {
    p.sko[i] = kp_strides[i];
    p.svo[i] = vp_strides[i];
  }
  p.pos = positions;
  p.pos64 = positions_64;
  p.sp[1] = pos_stride;
  p.inv_freq = inv_freq;
  p.tokens = tokens;
  p.S = 1;
  p.Hq = (int)num_q_heads;
  p.Hkv = (int)num_kv_heads;
  p.D = (int)head_dim;
  p.pairs = (int)(rotary_dim / 2);
  p.scale = scale;
  p.table = block_table;
  p.bt_stride = block_table_stride;
  p.kv_lens = kv_lens;
  p.cu = cu_seqlens;
  p.N = (int)num_seqs;
  p.ps_shift = __builtin_ctzll((unsigned long long)page_size);
  p.num_pages = (int)num_pages;
  p.cap = max_pages * page_size;
  p.slot_pos = slot_positions;
  const bool vec = whole_vectors(head_dim, rotary_dim, interleaved) && vector_rows(q, q_strides, 2) &&
                   vector_rows(k, k_strides, 2) && vector_rows(v, v_strides, 2) && vector_rows(q_out, qo_strides, 2) &&
                   vector_rows(k_pages, kp_strides, 3) && vector_rows(v_pages, vp_strides, 3);
  return launch_rotary<true>(p, vec, interleaved, dtype, (hipStream_t)stream, what);
}
