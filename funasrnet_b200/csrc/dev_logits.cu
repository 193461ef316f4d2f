// Penalties, biases and masks on logits, and the greedy pick (fa_dev_adjust_logits).
//
// Almost every logit only passes through: the history and the biases touch a few
// hundred tokens of a vocabulary.  So a CTA first marks those in a bitmap and
// gathers (token, times generated, last bias entry) in a hash table, both in
// shared memory and with integer atomics, so that the order of arrival cannot
// change a result; then it streams its part of the row, copying bits, writing
// -inf under the mask and keeping the largest unmarked value; then it computes
// the marked tokens, one thread each, in 32 bits (the result alone is rounded to
// the type, the pick comes before that).  Counts per token in shared memory, looked
// up for every logit, took twice as long: the tables held the stream up.  The
// CTAs of a row form a cluster and send their best (value, index) to the first.
// One launch, no scratch.
//
// Bound: the logits' bytes, read once and written once.  256 f32 rows of 151936
// take 72.5 us, 4.3 of the 6.5 TB/s that a copy reaches (the tables' latency at
// each row's start is not hidden by the SM's other CTA alone, and 256 rows leave 40
// SMs with half the work of the others); 64 bf16 rows, cut in two, 13.8 us; one row, cut in 16, 6.1 us, a chain of latencies: offsets, lists,
// atomics, logits, the cluster's best.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "dev_ops.h"
#include "dev_ptx.cuh"

namespace fa {

namespace cg = cooperative_groups;

namespace {

// 256 threads make every chain of a thread's work twice as long (256 rows 108 us), 1024 leave one CTA an SM (75).
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMaxCluster = 16;
// Rows that several CTAs share, and rows of one CTA: 16-byte groups per thread and
// iteration, and slots of the hash table.  A part of a row is over before more loads
// pay, and every slot is cleared and looked at: one row 6.1 us with 1 group and 512
// slots, 6.3 with 1024, 7.0 with 2 groups and 2048.  Whole rows need loads in flight:
// 256 rows 75.8, 72.5 and 75.3 us with 2, 3 and 4 groups (4 spill).
template <bool kCut>
struct Tuning {
  static constexpr int kUnroll = kCut ? 1 : 3, kLogSlots = kCut ? 9 : 11;
};
constexpr int kFetch = 2;      // history or bias entries that a thread has in flight
// CTAs from which a row is not cut further.  64 rows: 24.7 us uncut, 13.8 in halves, 14.2 in quarters.
constexpr int kWanted = 74;
constexpr int kMinSpan = 2048, kMaxSpan = 1 << 20;  // tokens of a CTA

void need(bool ok, const char* what) {
  if (!ok) throw Error(kErrArgument, what);
}

struct Best {
  float v;
  int i;
};
// The larger value, of equal ones the lower index; NaN and -inf never enter.
__device__ __forceinline__ Best pick(Best a, Best b) {
  return b.i >= 0 && (a.i < 0 || b.v > a.v || (b.v == a.v && b.i < a.i)) ? b : a;
}
__device__ __forceinline__ Best warp_best(Best b) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    Best o;
    o.v = __shfl_xor_sync(0xffffffffu, b.v, d);
    o.i = __shfl_xor_sync(0xffffffffu, b.i, d);
    b = pick(b, o);
  }
  return b;
}

__device__ __forceinline__ int clamp_off(int x, long long hi) { return (int)min((long long)max(x, 0), hi); }

// Writes `b` to `slot` of the cluster's first CTA and counts its bytes on that
// CTA's barrier.
__device__ __forceinline__ void send_best(Best b, Best* slot, uint64_t* bar) {
  asm volatile(
      "{\n .reg .b32 s, m;\n .reg .b64 v;\n mapa.shared::cluster.u32 s, %0, 0;\n mapa.shared::cluster.u32 m, %1, 0;\n"
      " mov.b64 v, {%2, %3};\n st.async.shared::cluster.mbarrier::complete_tx::bytes.b64 [s], v, [m];\n}\n" ::"r"(
          ptx::saddr(slot)),
      "r"(ptx::saddr(bar)), "r"(__float_as_uint(b.v)), "r"(b.i)
      : "memory");
}

constexpr int kLogitsWait = 51;  // error-word code of a best value that never came

// Entries i, i + kThreads, ... of a list that ends before i1; -1 behind it.
__device__ __forceinline__ void fetch(const int* list, int i, int i1, int* t) {
#pragma unroll
  for (int k = 0; k < kFetch; ++k) t[k] = i1 - i > k * kThreads ? list[i + k * kThreads] : -1;
}
// f(token, index) for the entries [i0, i1) of a list, by all threads of the CTA; t has the thread's first ones.
template <typename F>
__device__ __forceinline__ void for_entries(const int* list, int i0, int i1, int* t, F&& f) {
  for (int i = i0 + (int)threadIdx.x;;) {
#pragma unroll
    for (int k = 0; k < kFetch; ++k) f(t[k], i + k * kThreads);
    if (i1 - i <= kFetch * kThreads) break;
    i += kFetch * kThreads;
    fetch(list, i, i1, t);
  }
}

// The bits of tokens e .. last (fewer than 32) from 32-bit words whose first stands for tokens 32 * w0 on.
__device__ __forceinline__ unsigned bits_of(const unsigned* words, int w0, int e, int last) {
  return __funnelshift_r(words[(e >> 5) - w0], words[(last >> 5) - w0], e & 31);
}

template <typename T, bool kCut>
__global__ void __launch_bounds__(kThreads, 2) adjust_logits_kernel(const fa_logits_args a, int span, int* err) {
  constexpr int VE = 16 / sizeof(T), U = Tuning<kCut>::kUnroll, kSlots = 1 << Tuning<kCut>::kLogSlots, kStep = kThreads * VE;
  constexpr unsigned kFull = (1u << VE) - 1;
  extern __shared__ __align__(16) unsigned marks[];  // one bit per token of the part
  __shared__ int slot_token[kSlots];      // -1: free
  __shared__ unsigned slot_seen[kSlots];  // bit 31: in the prompt; below: times generated.  Then the new logit
  __shared__ int slot_bias[kSlots];       // last bias entry + 1
  __shared__ int overflow;
  __shared__ int before[kMaxSpan / 1024 + 1];  // marked tokens before each 1024 of the part
  __shared__ __align__(16) Best from[kMaxCluster * kWarps];  // the first CTA: every warp's best
  __shared__ uint64_t arrived;
  const int rank = (int)cg::this_cluster().block_rank(), ranks = (int)cg::this_cluster().num_blocks();
  const int row = blockIdx.x / ranks;
  const int lo = rank * span, hi = min(lo + span, a.vocab);  // this CTA's tokens; span is a multiple of 32

  const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride;
  T* out = static_cast<T*>(a.out) + row * a.out_stride;
  // Elements by which the row's start lies past a 16-byte boundary; vector
  // loads start on the boundaries, vector stores where out lies alike.
  const int skew = (int)((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T));
  const bool alike = (reinterpret_cast<uintptr_t>(out) & 15) / sizeof(T) == (unsigned)skew;
  const int first = (lo + skew) / VE * VE - skew + (int)threadIdx.x * VE;  // this thread's first group

  auto load = [&](int e) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (e >= lo && e + VE <= hi) {
      v = __ldcs(reinterpret_cast<const uint4*>(in + e));
    } else if (e < hi) {  // the part's ragged ends
      T* t = reinterpret_cast<T*>(&v);
#pragma unroll
      for (int i = 0; i < VE; ++i)
        if (e + i >= lo && e + i < hi) t[i] = in[e + i];
    }
    return v;
  };
  uint4 v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) v[u] = load(first + u * kStep);

  if (ranks > 1 && a.tokens) {
    if (threadIdx.x == 0) {
      ptx::mbar_init(&arrived, 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      ptx::mbar_expect_tx(&arrived, (unsigned)(ranks * kWarps * sizeof(Best)));
    }
    ptx::cluster_arrive();
  }
  int h0 = 0, made = 0, h1 = 0, b0 = 0, b1 = 0;  // prompt [h0, made), generated [made, h1), biases [b0, b1)
  if (a.history) {
    h0 = clamp_off(a.history_offsets[row], a.history_total);
    h1 = clamp_off(a.history_offsets[row + 1], a.history_total);
    if (a.prompt_lens) made = max(min(a.prompt_lens[row], h1 - h0), 0);
    made += h0;
  }
  if (a.bias_tokens) {
    b0 = clamp_off(a.bias_offsets[row], a.bias_total);
    b1 = clamp_off(a.bias_offsets[row + 1], a.bias_total);
  }
  const uint32_t* mask = nullptr;
  if (a.mask) {
    const int r = a.mask_rows ? a.mask_rows[row] : row;
    if (r >= 0 && r < a.mask_count) mask = a.mask + r * a.mask_stride;
  }
  const bool marked = h1 > h0 || b1 > b0;
  const float rep = a.repetition ? a.repetition[row] : 1.0f;
  const float pres = a.presence ? a.presence[row] : 0.0f;
  const float freq = a.frequency ? a.frequency[row] : 0.0f;

  auto clear = [&] {
    for (int s = threadIdx.x; s < kSlots; s += kThreads) {
      slot_token[s] = -1;
      slot_seen[s] = 0;
      slot_bias[s] = 0;
    }
  };
  // A marked token's number among the marked ones.
  auto rank_of = [&](int t) {
    const int w = (t - lo) >> 5;
    int n = before[w >> 5] + __popc(marks[w] & ((1u << (t & 31)) - 1));
    for (int i = w & ~31; i < w; ++i) n += __popc(marks[i]);
    return n;
  };
  // Gathers the entries of this part's tokens into the slots: by hash, marking the
  // tokens, or (kRanked) those of the marked tokens from number r0 on.
  auto gather = [&](auto ranked, int r0, int* seen_t, int* bias_t) {
    constexpr bool kRanked = decltype(ranked)::value;
    const unsigned n = hi - lo;
    auto slot_of = [&](int t) {
      if (kRanked) {
        const int r = rank_of(t) - r0;
        if ((unsigned)r >= (unsigned)kSlots) return -1;
        slot_token[r] = t;
        return r;
      }
      atomicOr(&marks[(t - lo) >> 5], 1u << (t & 31));
      int s = (int)((unsigned)t * 2654435761u >> (32 - Tuning<kCut>::kLogSlots));  // multiplicative hash
      for (int probe = 0; probe < 32; ++probe, s = (s + 1) & (kSlots - 1)) {
        const int before = atomicCAS(&slot_token[s], -1, t);
        if (before == -1 || before == t) return s;
      }
      overflow = 1;
      return -1;
    };
    for_entries(a.history, h0, h1, seen_t, [&](int t, int i) {
      if ((unsigned)(t - lo) >= n) return;
      const int s = slot_of(t);
      if (s < 0) return;
      if (i < made) atomicOr(&slot_seen[s], 0x80000000u);
      else atomicAdd(&slot_seen[s], 1u);
    });
    for_entries(a.bias_tokens, b0, b1, bias_t, [&](int t, int i) {
      if ((unsigned)(t - lo) >= n) return;
      const int s = slot_of(t);
      if (s >= 0) atomicMax(&slot_bias[s], i - b0 + 1);
    });
  };
  // The new logits of this thread's slots, in the place of what the slots counted.
  auto compute = [&](const T* from_row) {
    constexpr int K = kSlots / kThreads;
    float x[K], bias[K];
    unsigned allowed[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int s = threadIdx.x + k * kThreads, t = slot_token[s], b = slot_bias[s];
      x[k] = t < 0 ? 0.0f : (float)from_row[t];
      bias[k] = t < 0 || b == 0 ? 0.0f : a.bias_values[b0 + b - 1];
      allowed[k] = t < 0 || mask == nullptr ? 1u : mask[t >> 5] >> (t & 31);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int s = threadIdx.x + k * kThreads;
      const unsigned seen = slot_seen[s], n = seen & 0x7fffffffu;
      float y = x[k];
      if (seen != 0) y = y > 0.0f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
      if (n != 0) y = __fsub_rn(y, __fadd_rn(__fmul_rn(freq, (float)n), pres));
      if (slot_bias[s] != 0) y = __fadd_rn(y, bias[k]);
      slot_seen[s] = __float_as_uint(allowed[k] & 1u ? y : -INFINITY);
    }
  };
  if (a.history || a.bias_tokens) {  // under the latency of the offsets
    clear();
    for (int i = threadIdx.x; i < span / 32; i += kThreads) marks[i] = 0;
    if (threadIdx.x == 0) overflow = 0;
  }
  int seen_t[kFetch], bias_t[kFetch];
  auto fetch_first = [&] {
    fetch(a.history, h0 + (int)threadIdx.x, h1, seen_t);
    fetch(a.bias_tokens, b0 + (int)threadIdx.x, b1, bias_t);
  };
  if (marked) {
    fetch_first();
    __syncthreads();
    gather(std::false_type{}, 0, seen_t, bias_t);
    __syncthreads();
    if (!overflow) compute(in);  // their logits' latency passes with the stream's first
  }

  // ---- the stream ----
  Best best{-INFINITY, -1};
  for (int e0 = first; e0 < hi; e0 += U * kStep) {
    uint4 next[U];
#pragma unroll
    for (int u = 0; u < U; ++u) next[u] = load(e0 + (U + u) * kStep);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = e0 + u * kStep;
      if (e >= hi) break;
      const bool whole = e >= lo && e + VE <= hi;
      const int from_e = max(e, lo), last = min(e + VE, hi) - 1;
      unsigned keep = ~0u, open = ~0u;  // elements that stay as they are; that may be the largest
      if (!whole) open = (kFull << (from_e - e)) & (kFull >> (e + VE - 1 - last));
      if (mask) {
        keep = bits_of(mask, 0, from_e, last) << (from_e - e);
        open &= keep;
      }
      if (marked) {
        const unsigned m = bits_of(marks, lo >> 5, from_e, last) << (from_e - e);
        keep |= m;
        open &= ~m;
      }
      T* t = reinterpret_cast<T*>(&v[u]);
      float x[VE];
#pragma unroll
      for (int i = 0; i < VE; ++i) x[i] = (float)t[i];
      if ((open & kFull) != kFull) {
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          if (!((open >> i) & 1u)) x[i] = -INFINITY;
          if (!((keep >> i) & 1u)) t[i] = T(-INFINITY);
        }
      }
      float top = x[0];
#pragma unroll
      for (int i = 1; i < VE; ++i) top = fmaxf(top, x[i]);
      if (top > best.v) {
        best.v = top;
#pragma unroll
        for (int i = VE - 1; i >= 0; --i)
          if (x[i] == top) best.i = e + i;
      }
      if (alike && whole) {
        __stcs(reinterpret_cast<uint4*>(out + e), v[u]);
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i)
          if (e + i >= lo && e + i < hi) out[e + i] = t[i];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = next[u];
  }

  // ---- the marked tokens, whose logits the stream left as they were ----
  if (marked) {
    auto finish = [&] {
#pragma unroll
      for (int k = 0; k < kSlots / kThreads; ++k) {
        const int s = threadIdx.x + k * kThreads, t = slot_token[s];
        if (t < 0) continue;
        const float x = __uint_as_float(slot_seen[s]);
        if (x > best.v || (x == best.v && best.i >= 0 && t < best.i)) best = Best{x, t};
        out[t] = (T)x;
      }
    };
    __syncthreads();
    if (!overflow) {
      finish();
    } else {  // more tokens than slots: kSlots of them at a time
      const int lane = threadIdx.x & 31, blocks = (hi - lo + 1023) / 1024;
      for (int b = threadIdx.x >> 5; b < blocks; b += kWarps) {
        const int w = b * 32 + lane, n = __reduce_add_sync(0xffffffffu, w < span / 32 ? __popc(marks[w]) : 0);
        if (lane == 0) before[b] = n;
      }
      __syncthreads();
      if (threadIdx.x < 32) {
        int sum = 0;
        for (int b = lane; b - lane < blocks; b += 32) {
          const int n = b < blocks ? before[b] : 0;
          int upto = n;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += x;
          }
          if (b < blocks) before[b] = sum + upto - n;
          sum += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (lane == 0) before[blocks] = sum;
      }
      __syncthreads();
      for (int r0 = 0, all = before[blocks]; r0 < all; r0 += kSlots) {
        __syncthreads();
        clear();
        fetch_first();
        __syncthreads();
        gather(std::true_type{}, r0, seen_t, bias_t);
        __syncthreads();
        compute(out);
        finish();
      }
    }
  }
  if (a.tokens == nullptr) return;
  const int warp = threadIdx.x >> 5;
  best = warp_best(best);
  if (ranks == 1) {
    if ((threadIdx.x & 31) == 0) from[warp] = best;
    __syncthreads();
    if (warp != 0) return;
  } else {
    ptx::cluster_wait();  // the first CTA's barrier is ready since its start
    if ((threadIdx.x & 31) == 0) send_best(best, &from[rank * kWarps + warp], &arrived);
    if (rank != 0 || warp != 0) return;
    // The copies are on their way from CTAs that wait for nothing: bounded all the same (4 us a try: about a minute).
    bool here = false;
    for (int i = 0; i < (1 << 24) && !here; ++i) here = ptx::mbar_try_wait(&arrived, 0);
    here = __all_sync(0xffffffffu, here);
    if (!here) {
      if (threadIdx.x == 0) atomicCAS(err, 0, kLogitsWait);
      return;
    }
  }
  best = Best{-INFINITY, -1};
  for (int i = threadIdx.x; i < ranks * kWarps; i += 32) best = pick(best, from[i]);
  best = warp_best(best);
  if (threadIdx.x == 0) a.tokens[row] = best.i;
}

template <typename T>
void launch(const fa_logits_args& a, int* err, cudaStream_t stream) {
  int ranks = 1;
  while (ranks < kMaxCluster && (a.rows * (int64_t)ranks < kWanted || a.vocab > ranks * kMaxSpan) &&
         a.vocab > ranks * kMinSpan)
    ranks *= 2;
  const int span = ((a.vocab + ranks - 1) / ranks + 31) / 32 * 32;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = (unsigned)a.rows * ranks;
  cfg.blockDim = kThreads;
  cfg.dynamicSmemBytes = a.history || a.bias_tokens ? span / 8 : 0;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ranks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  FA_CUDA(cudaLaunchKernelEx(&cfg, ranks > 1 ? adjust_logits_kernel<T, true> : adjust_logits_kernel<T, false>, a, span, err));
}

template <typename T, bool kCut>
void prepare() {
  FA_CUDA(cudaFuncSetAttribute(adjust_logits_kernel<T, kCut>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               FA_LOGITS_MAX_VOCAB / kMaxCluster / 8));
  FA_CUDA(cudaFuncSetAttribute(adjust_logits_kernel<T, kCut>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
}

}  // namespace

void prepare_dev_logits() {
  prepare<float, true>();
  prepare<float, false>();
  prepare<__half, true>();
  prepare<__half, false>();
  prepare<__nv_bfloat16, true>();
  prepare<__nv_bfloat16, false>();
}

int check_logits(const fa_logits_args* a) {
  need(a != nullptr, "null arguments");
  need(a->dtype == FA_DTYPE_F32 || a->dtype == FA_DTYPE_F16 || a->dtype == FA_DTYPE_BF16, "unknown dtype");
  need(a->rows >= 0 && a->vocab >= 1 && a->mask_count >= 0, "negative rows or mask_count, or vocab below one");
  need(a->history_total >= 0 && a->history_total < (1ll << 31) && a->bias_total >= 0 && a->bias_total < (1ll << 31),
       "history_total or bias_total is negative or beyond 2^31");
  if (a->vocab > FA_LOGITS_MAX_VOCAB || a->rows > (1 << 27)) return kDeclined;
  if (a->rows == 0) return kHandled;
  need(a->logits && a->out, "null logits or out");
  need(aligned_to(a->dtype == FA_DTYPE_F32 ? 4 : 2, {a->logits, a->out}), "logits or out not aligned to their type");
  need(aligned_to(4, {a->tokens, a->history, a->history_offsets, a->prompt_lens, a->repetition, a->presence, a->frequency,
                      a->bias_tokens, a->bias_values, a->bias_offsets, a->mask, a->mask_rows}),
       "an array not aligned to 4 bytes");
  const int64_t far = 1ll << 34;
  need(a->logits_stride >= 0 && a->out_stride >= 0 && a->mask_stride >= 0, "negative stride");
  need(a->rows == 1 || (a->logits_stride < far && a->out_stride < far), "a stride is beyond 2^34 elements");
  need(a->rows == 1 || (a->logits_stride >= a->vocab && a->out_stride >= a->vocab), "rows overlap: stride below vocab");
  // In place, or apart: rows of out on other rows of the logits would be read changed.
  const int64_t size = a->dtype == FA_DTYPE_F32 ? 4 : 2;
  const uintptr_t x = reinterpret_cast<uintptr_t>(a->logits), y = reinterpret_cast<uintptr_t>(a->out);
  const uint64_t xn = ((a->rows - 1) * a->logits_stride + a->vocab) * size, yn = ((a->rows - 1) * a->out_stride + a->vocab) * size;
  bool apart = x + xn <= y || y + yn <= x;
  if (!apart && a->rows > 1 && a->logits_stride == a->out_stride) {  // columns of one array side by side
    const int64_t stride = a->logits_stride * size, off = ((int64_t)(y - x) % stride + stride) % stride;
    apart = off >= a->vocab * size && stride - off >= a->vocab * size;
  }
  need(apart || (x == y && (a->rows == 1 || a->logits_stride == a->out_stride)),
       "out overlaps logits and is not the same rows");
  need(!a->history || a->history_offsets, "history without history_offsets");
  need(!a->bias_tokens || (a->bias_values && a->bias_offsets), "bias_tokens without bias_values or bias_offsets");
  need(!a->mask || a->mask_stride >= (a->vocab + 31) / 32 || a->mask_count <= 1, "mask rows overlap");
  need(!a->mask || a->mask_rows || a->mask_count >= a->rows, "fewer mask rows than rows, and no mask_rows");
  return kHandled;
}

void launch_adjust_logits(const fa_logits_args& a, int* err, cudaStream_t stream) {
  if (a.rows == 0) return;
  if (a.dtype == FA_DTYPE_F32)
    launch<float>(a, err, stream);
  else if (a.dtype == FA_DTYPE_F16)
    launch<__half>(a, err, stream);
  else
    launch<__nv_bfloat16>(a, err, stream);
}

}  // namespace fa
