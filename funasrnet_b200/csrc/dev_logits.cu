// Penalties, biases and masks on logits, and the greedy pick (fa_dev_adjust_logits).
//
// One thread-block cluster per row.  Its CTAs share the vocabulary in windows;
// a CTA counts the row's history over its window in shared memory (integer
// atomics, so the order of arrival cannot change a result), then streams the
// window's logits once: read, change, write, and keep the best (value, index).
// The cluster's CTAs hand their best to the first one through distributed
// shared memory.  Bound: the logits' bytes, read once and written once.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "dev_ops.h"

namespace fa {

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 512;
constexpr int kCluster = 8;        // CTAs per row
constexpr int kWindow = 8192;      // tokens per window at most (two words of shared memory each)

void need(bool ok, const char* what) {
  if (!ok) throw Error(kErrArgument, what);
}

template <typename T>
__device__ __forceinline__ float to_f32(T v) { return (float)v; }

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

__device__ __forceinline__ long long clamp_off(int x, long long hi) { return min((long long)max(x, 0), hi); }

template <typename T>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads)
    adjust_logits_kernel(const fa_logits_args a, int window, int windows) {
  extern __shared__ unsigned sm_words[];
  unsigned* seen = sm_words;                          // bit 31: in the history; below: times generated
  int* bias_at = reinterpret_cast<int*>(sm_words + (a.history ? window : 0));  // last bias entry + 1
  __shared__ Best part[kThreads / 32];
  __shared__ Best mine;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank();
  const int row = blockIdx.x / kCluster;
  constexpr int VE = 16 / sizeof(T);

  const float rep = a.repetition ? a.repetition[row] : 1.0f;
  const float pres = a.presence ? a.presence[row] : 0.0f;
  const float freq = a.frequency ? a.frequency[row] : 0.0f;
  long long h0 = 0, h1 = 0, made = 0, b0 = 0, b1 = 0;
  if (a.history) {
    h0 = clamp_off(a.history_offsets[row], a.history_total);
    h1 = clamp_off(a.history_offsets[row + 1], a.history_total);
    made = h0 + (a.prompt_lens ? max(a.prompt_lens[row], 0) : 0);
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
  const T* in = static_cast<const T*>(a.logits) + row * a.logits_stride;
  T* out = static_cast<T*>(a.out) + row * a.out_stride;
  // Elements by which the row's start lies past a 16-byte boundary; vector
  // loads start on the boundaries, vector stores where out lies alike.
  const int skew = (int)((reinterpret_cast<uintptr_t>(in) & 15) / sizeof(T));
  const bool alike = (reinterpret_cast<uintptr_t>(out) & 15) / sizeof(T) == (unsigned)skew;

  Best best{-INFINITY, -1};
  for (int w = rank; w < windows; w += kCluster) {
    const int lo = w * window, hi = min(lo + window, a.vocab);
    __syncthreads();
    if (a.history)
      for (int i = threadIdx.x; i < window; i += kThreads) seen[i] = 0;
    if (a.bias_tokens)
      for (int i = threadIdx.x; i < window; i += kThreads) bias_at[i] = 0;
    __syncthreads();
    for (long long i = h0 + threadIdx.x; i < h1; i += kThreads) {
      const int t = a.history[i];
      if (t >= lo && t < hi) {
        atomicOr(&seen[t - lo], 0x80000000u);
        if (i >= made) atomicAdd(&seen[t - lo], 1u);
      }
    }
    for (long long i = b0 + threadIdx.x; i < b1; i += kThreads) {
      const int t = a.bias_tokens[i];
      if (t >= lo && t < hi) atomicMax(&bias_at[t - lo], (int)(i - b0) + 1);
    }
    __syncthreads();
    const int groups = (hi - lo + skew + VE - 1 + (lo % VE)) / VE + 1;
    const int first = (lo + skew) / VE * VE - skew;  // <= lo, on a boundary
    for (int g = threadIdx.x; g < groups; g += kThreads) {
      const int e0 = first + g * VE;
      if (e0 >= hi) break;
      const bool whole = e0 >= lo && e0 + VE <= hi;
      T v[VE];
      if (whole) {
        *reinterpret_cast<uint4*>(v) = __ldcs(reinterpret_cast<const uint4*>(in + e0));
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i)
          if (e0 + i >= lo && e0 + i < hi) v[i] = in[e0 + i];
      }
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const int t = e0 + i;
        if (t < lo || t >= hi) continue;
        float x = to_f32(v[i]);
        if (a.history) {
          const unsigned s = seen[t - lo];
          if (s != 0) {
            x = x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
            const unsigned n = s & 0x7fffffffu;
            if (n != 0) x = __fsub_rn(x, __fadd_rn(__fmul_rn(freq, (float)n), pres));
          }
        }
        if (a.bias_tokens) {
          const int at = bias_at[t - lo];
          if (at != 0) x = __fadd_rn(x, a.bias_values[b0 + at - 1]);
        }
        if (mask && !((mask[t >> 5] >> (t & 31)) & 1u)) x = -INFINITY;
        if (x > best.v) best = Best{x, t};
        v[i] = (T)x;
      }
      if (whole && alike) {
        __stcs(reinterpret_cast<uint4*>(out + e0), *reinterpret_cast<const uint4*>(v));
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i)
          if (e0 + i >= lo && e0 + i < hi) out[e0 + i] = v[i];
      }
    }
  }
  best = warp_best(best);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = best;
  __syncthreads();
  if (threadIdx.x < 32) {
    best = threadIdx.x < kThreads / 32 ? part[threadIdx.x] : Best{-INFINITY, -1};
    best = warp_best(best);
    if (threadIdx.x == 0) mine = best;
  }
  cluster.sync();
  if (rank == 0 && threadIdx.x < 32) {
    best = threadIdx.x < kCluster ? *cluster.map_shared_rank(&mine, (int)threadIdx.x) : Best{-INFINITY, -1};
    best = warp_best(best);
    if (threadIdx.x == 0 && a.tokens) a.tokens[row] = best.i;
  }
  cluster.sync();  // the others' shared memory stays until it was read
}

template <typename T>
void launch(const fa_logits_args& a, cudaStream_t stream) {
  const int rounds = (a.vocab + kCluster * kWindow - 1) / (kCluster * kWindow);
  int window = (a.vocab + kCluster * rounds - 1) / (kCluster * rounds);
  window = (window + 127) / 128 * 128;
  const int windows = (a.vocab + window - 1) / window;
  const int words = (a.history ? window : 0) + (a.bias_tokens ? window : 0);
  FA_CUDA(cudaFuncSetAttribute(adjust_logits_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * 4 * kWindow));
  adjust_logits_kernel<T><<<(unsigned)a.rows * kCluster, kThreads, words * 4, stream>>>(a, window, windows);
  FA_CUDA(cudaGetLastError());
}

}  // namespace

int check_logits(const fa_logits_args* a) {
  need(a != nullptr, "null arguments");
  need(a->dtype == FA_DTYPE_F32 || a->dtype == FA_DTYPE_F16 || a->dtype == FA_DTYPE_BF16, "unknown dtype");
  need(a->rows >= 0 && a->vocab >= 1 && a->mask_count >= 0, "negative rows or mask_count, or vocab below one");
  need(a->history_total >= 0 && a->history_total < (1ll << 31) && a->bias_total >= 0 && a->bias_total < (1ll << 31),
       "history_total or bias_total is negative or beyond 2^31");
  if (a->vocab > FA_LOGITS_MAX_VOCAB || a->rows > (1 << 27)) return kDeclined;
  if (a->rows == 0) return kHandled;
  need(a->logits && a->out, "null logits or out");
  need(a->rows == 1 || (a->logits_stride >= a->vocab && a->out_stride >= a->vocab), "rows overlap: stride below vocab");
  need(a->logits_stride >= 0 && a->out_stride >= 0 && a->mask_stride >= 0, "negative stride");
  need(!a->history || a->history_offsets, "history without history_offsets");
  need(!a->bias_tokens || (a->bias_values && a->bias_offsets), "bias_tokens without bias_values or bias_offsets");
  need(!a->mask || a->mask_stride >= (a->vocab + 31) / 32 || a->mask_count <= 1, "mask rows overlap");
  need(!a->mask || a->mask_rows || a->mask_count >= a->rows, "fewer mask rows than rows, and no mask_rows");
  return kHandled;
}

void launch_adjust_logits(const fa_logits_args& a, cudaStream_t stream) {
  if (a.rows == 0) return;
  if (a.dtype == FA_DTYPE_F32)
    launch<float>(a, stream);
  else if (a.dtype == FA_DTYPE_F16)
    launch<__half>(a, stream);
  else
    launch<__nv_bfloat16>(a, stream);
}

}  // namespace fa
