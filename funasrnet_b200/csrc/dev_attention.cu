// Attention over packed sequences and over a shared prefix (fa_dev_attention_*).
//
//     out_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_i . k_j - m_i)
//
// over the keys j that query i sees, in one pass with the running maximum m_i.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "dev_ops.h"

namespace fa {

namespace {

__device__ int g_dev_error;

// ------------------------------------------------------------- checks ----

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

void need(bool ok, const char* what) {
  if (!ok) throw Error(kErrArgument, what);
}

// Strides in elements of two bytes: every row must start on 16 bytes.
bool strides16(const int64_t* s, int n) {
  for (int i = 0; i < n; ++i)
    if (s[i] % 8 != 0) return false;
  return true;
}

void need_strides(const int64_t* s, int n) {
  for (int i = 0; i < n; ++i) need(s[i] >= 0 && s[i] < (1ll << 38), "a stride is negative or beyond 2^38 elements");
}

void check_heads(int dtype, int sequences, int heads, int kv_heads, int head_size, float scale) {
  need(dtype == FA_DTYPE_F32 || dtype == FA_DTYPE_F16 || dtype == FA_DTYPE_BF16, "unknown dtype");
  need(sequences >= 0, "negative sequence count");
  need(heads >= 1 && kv_heads >= 1 && head_size >= 1, "heads, kv_heads and head_size must be positive");
  need(heads % kv_heads == 0, "heads must be a multiple of kv_heads");
  need(std::isfinite(scale), "scale must be finite");
}

bool heads_supported(int dtype, int heads, int kv_heads, int head_size) {
  return dtype != FA_DTYPE_F32 && head_size % 8 == 0 && head_size <= 128 && heads / kv_heads <= 64;
}

// ------------------------------------------------------------ kernels ----

template <typename T>
__device__ __forceinline__ void load4(const T* p, float* v) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (float)t[i];
}

struct KvRun {
  const void *k, *v;
  long long k_row, v_row;  // element strides between keys
  int n;                   // keys
};

// One warp: one query head over up to two runs of keys, lane l holding the
// channels 4l .. 4l + 3.
template <typename T>
__device__ __forceinline__ void attend_row(const T* q, const KvRun* runs, int n_runs, int head_size, float scale, T* out,
                                           float* lse) {
  const int lane = threadIdx.x & 31, c = lane * 4;
  const bool on = c < head_size;
  float qv[4] = {}, o[4] = {};
  if (on) load4(q + c, qv);
  float m = -INFINITY, l = 0.0f;
  for (int r = 0; r < n_runs; ++r) {
    for (int j = 0; j < runs[r].n; ++j) {
      float kv[4] = {}, vv[4] = {};
      if (on) {
        load4(static_cast<const T*>(runs[r].k) + j * runs[r].k_row + c, kv);
        load4(static_cast<const T*>(runs[r].v) + j * runs[r].v_row + c, vv);
      }
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) s = fmaf(qv[i], kv[i], s);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      s *= scale;
      const float top = fmaxf(m, s), base = top == -INFINITY ? 0.0f : top;
      const float f = expf(m - base), p = expf(s - base);
      m = top;
      l = l * f + p;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = o[i] * f + p * vv[i];
    }
  }
  if (on) {
    T t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = (T)(l == 0.0f ? 0.0f : o[i] / l);
    *reinterpret_cast<uint2*>(out + c) = *reinterpret_cast<const uint2*>(t);
  }
  if (lse && lane == 0) *lse = (m == -INFINITY ? 0.0f : m) + logf(l);
}

// The sequence that holds row t: the last b with off[b] <= t.
__device__ __forceinline__ int find_sequence(const int* off, int n, long long t) {
  int lo = 0, hi = n;  // off[lo] <= t < off[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (off[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int clamp_to(int x, long long hi) { return (int)min((long long)max(x, 0), hi); }

template <typename T>
__global__ void __launch_bounds__(128) packed_rows_kernel(const fa_attention_packed_args a) {
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const long long t = row / a.heads;
  const int h = (int)(row - t * a.heads);
  if (t >= a.total_q || t < a.q_offsets[0] || t >= a.q_offsets[a.sequences]) return;
  const int b = find_sequence(a.q_offsets, a.sequences, t);
  const int q0 = clamp_to(a.q_offsets[b], a.total_q), q1 = clamp_to(a.q_offsets[b + 1], a.total_q);
  const int k0 = clamp_to(a.k_offsets[b], a.total_k), k1 = clamp_to(a.k_offsets[b + 1], a.total_k);
  int n = max(k1 - k0, 0);
  if (a.causal) n = max(0, min(n, (int)(t - q0) + n - (q1 - q0) + 1));
  const int kh = h / (a.heads / a.kv_heads);
  KvRun run;
  run.k = static_cast<const T*>(a.k) + k0 * a.k_stride[0] + kh * a.k_stride[1];
  run.v = static_cast<const T*>(a.v) + k0 * a.v_stride[0] + kh * a.v_stride[1];
  run.k_row = a.k_stride[0];
  run.v_row = a.v_stride[0];
  run.n = n;
  attend_row<T>(static_cast<const T*>(a.q) + t * a.q_stride[0] + h * a.q_stride[1], &run, 1, a.head_size, a.scale,
                static_cast<T*>(a.out) + t * a.out_stride[0] + h * a.out_stride[1], a.lse ? a.lse + row : nullptr);
}

template <typename T>
__global__ void __launch_bounds__(128) shared_rows_kernel(const fa_attention_shared_args a) {
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const long long b = row / a.heads;
  const int h = (int)(row - b * a.heads);
  if (b >= a.sequences) return;
  const int kh = h / (a.heads / a.kv_heads);
  KvRun run[2];
  run[0].k = static_cast<const T*>(a.prefix_k) + kh * a.prefix_k_stride[1];
  run[0].v = static_cast<const T*>(a.prefix_v) + kh * a.prefix_v_stride[1];
  run[0].k_row = a.prefix_k_stride[0];
  run[0].v_row = a.prefix_v_stride[0];
  run[0].n = (int)a.prefix_len;
  run[1].k = static_cast<const T*>(a.suffix_k) + b * a.suffix_k_stride[0] + kh * a.suffix_k_stride[2];
  run[1].v = static_cast<const T*>(a.suffix_v) + b * a.suffix_v_stride[0] + kh * a.suffix_v_stride[2];
  run[1].k_row = a.suffix_k_stride[1];
  run[1].v_row = a.suffix_v_stride[1];
  run[1].n = a.suffix_lens ? clamp_to(a.suffix_lens[b], a.suffix_capacity) : 0;
  attend_row<T>(static_cast<const T*>(a.q) + b * a.q_stride[0] + h * a.q_stride[1], run, 2, a.head_size, a.scale,
                static_cast<T*>(a.out) + b * a.out_stride[0] + h * a.out_stride[1], a.lse ? a.lse + row : nullptr);
}

}  // namespace

int check_attention_packed(const fa_attention_packed_args* a) {
  need(a != nullptr, "null arguments");
  check_heads(a->dtype, a->sequences, a->heads, a->kv_heads, a->head_size, a->scale);
  need(a->total_q >= 0 && a->total_k >= 0 && a->reserved == 0, "negative total or a reserved field that is not 0");
  need_strides(a->q_stride, 2);
  need_strides(a->k_stride, 2);
  need_strides(a->v_stride, 2);
  need_strides(a->out_stride, 2);
  if (!heads_supported(a->dtype, a->heads, a->kv_heads, a->head_size)) return kDeclined;
  if (a->total_q * a->heads >= (1ll << 31) || a->total_k >= (1ll << 31)) return kDeclined;
  if (a->total_q == 0 || a->sequences == 0) return kHandled;
  need(a->q && a->out && a->q_offsets && a->k_offsets, "null q, out, q_offsets or k_offsets");
  need(a->total_k == 0 || (a->k && a->v), "null k or v");
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out)) return kDeclined;
  if (!strides16(a->q_stride, 2) || !strides16(a->k_stride, 2) || !strides16(a->v_stride, 2) ||
      !strides16(a->out_stride, 2))
    return kDeclined;
  need(a->workspace_bytes >= attention_packed_workspace(a->total_q, a->total_k, a->sequences, a->heads, a->kv_heads,
                                                        a->head_size) &&
           (a->workspace_bytes == 0 || (a->workspace && aligned16(a->workspace))),
       "workspace smaller than fa_dev_attention_packed_workspace, or not on 16 bytes");
  return kHandled;
}

int check_attention_shared(const fa_attention_shared_args* a) {
  need(a != nullptr, "null arguments");
  check_heads(a->dtype, a->sequences, a->heads, a->kv_heads, a->head_size, a->scale);
  need(a->prefix_len >= 0 && a->suffix_capacity >= 0, "negative length");
  need_strides(a->q_stride, 2);
  need_strides(a->prefix_k_stride, 2);
  need_strides(a->prefix_v_stride, 2);
  need_strides(a->suffix_k_stride, 3);
  need_strides(a->suffix_v_stride, 3);
  need_strides(a->out_stride, 2);
  if (!heads_supported(a->dtype, a->heads, a->kv_heads, a->head_size)) return kDeclined;
  if ((int64_t)a->sequences * a->heads >= (1ll << 31) || a->prefix_len + a->suffix_capacity >= (1ll << 31))
    return kDeclined;
  if (a->sequences == 0) return kHandled;
  need(a->q && a->out, "null q or out");
  need(a->prefix_len == 0 || (a->prefix_k && a->prefix_v), "null prefix_k or prefix_v");
  need(a->suffix_capacity == 0 || (a->suffix_k && a->suffix_v && a->suffix_lens),
       "null suffix_k, suffix_v or suffix_lens");
  if (!aligned16(a->q) || !aligned16(a->prefix_k) || !aligned16(a->prefix_v) || !aligned16(a->suffix_k) ||
      !aligned16(a->suffix_v) || !aligned16(a->out))
    return kDeclined;
  if (!strides16(a->q_stride, 2) || !strides16(a->prefix_k_stride, 2) || !strides16(a->prefix_v_stride, 2) ||
      !strides16(a->suffix_k_stride, 3) || !strides16(a->suffix_v_stride, 3) || !strides16(a->out_stride, 2))
    return kDeclined;
  need(a->workspace_bytes >= attention_shared_workspace(a->prefix_len, a->suffix_capacity, a->sequences, a->heads,
                                                        a->kv_heads, a->head_size) &&
           (a->workspace_bytes == 0 || (a->workspace && aligned16(a->workspace))),
       "workspace smaller than fa_dev_attention_shared_workspace, or not on 16 bytes");
  return kHandled;
}

int64_t attention_packed_workspace(int64_t, int64_t, int, int, int, int) { return 0; }
int64_t attention_shared_workspace(int64_t, int64_t, int, int, int, int) { return 0; }

void launch_attention_packed(const fa_attention_packed_args& a, cudaStream_t stream) {
  if (a.total_q == 0 || a.sequences == 0) return;
  const unsigned grid = (unsigned)((a.total_q * a.heads + 3) / 4);
  if (a.dtype == FA_DTYPE_F16)
    packed_rows_kernel<__half><<<grid, 128, 0, stream>>>(a);
  else
    packed_rows_kernel<__nv_bfloat16><<<grid, 128, 0, stream>>>(a);
  FA_CUDA(cudaGetLastError());
}

void launch_attention_shared(const fa_attention_shared_args& a, cudaStream_t stream) {
  if (a.sequences == 0) return;
  const unsigned grid = (unsigned)(((int64_t)a.sequences * a.heads + 3) / 4);
  fa_attention_shared_args s = a;
  if (a.suffix_capacity == 0) s.suffix_lens = nullptr;
  if (a.dtype == FA_DTYPE_F16)
    shared_rows_kernel<__half><<<grid, 128, 0, stream>>>(s);
  else
    shared_rows_kernel<__nv_bfloat16><<<grid, 128, 0, stream>>>(s);
  FA_CUDA(cudaGetLastError());
}

int take_device_error() {
  FA_CUDA(cudaDeviceSynchronize());
  int code = 0;
  FA_CUDA(cudaMemcpyFromSymbol(&code, g_dev_error, sizeof(code)));
  const int zero = 0;
  if (code != 0) FA_CUDA(cudaMemcpyToSymbol(g_dev_error, &zero, sizeof(zero)));
  return code;
}

}  // namespace fa
