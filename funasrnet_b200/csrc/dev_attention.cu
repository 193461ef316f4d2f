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
#include "dev_ptx.cuh"
#include "tma_host.h"

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
  need(std::isfinite(scale) && scale > 0.0f, "scale must be positive and finite");
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

__device__ __forceinline__ int clamp_to(int x, long long hi) { return (int)min((long long)max(x, 0), hi); }

// -------------------------------------------------- tensor-core attention ----

constexpr int kRows = 128;     // query rows of one tile (TMEM lanes): tokens x heads of a KV head's group
constexpr int kKeys = 128;     // keys per step
constexpr float kSlack = 8.0f; // powers of two by which a row's maximum may rise before its sums are rescaled

enum AttnError : int { kAttnWaitLoad = 41, kAttnWaitMma = 42, kAttnWaitSoftmax = 43, kAttnWaitFree = 44 };

struct TcArgs {
  const int* q_off = nullptr;  // null: one sequence of all rows
  const int* k_off = nullptr;
  int sequences = 1;
  long long total_q = 0, total_k = 0;
  int heads = 0, kv_heads = 0, group = 0, head_size = 0;
  int tokens = 0;              // query tokens of a tile: kRows / group
  int tiles = 0;               // tile pairs of the whole call, an upper bound
  int splits = 1;
  int causal = 0;
  float scale = 0.0f, scale_log2 = 0.0f;
  void* out = nullptr;
  long long out_token = 0, out_head = 0;
  float* lse = nullptr;
  float* part_o = nullptr;     // splits > 1: [splits x total_q x heads x head_size], and the rows' lse
  float* part_lse = nullptr;
  int* err = nullptr;
};
struct TcMaps {
  CUtensorMap q;  // (channel, head of the group, KV head, token)
  CUtensorMap k;  // (channel, KV head, key)
  CUtensorMap v;
};

template <int D>
struct TcLayout {
  static constexpr int kHalf = kRows * 128;       // 128 rows x 64 channels, 128-byte swizzle
  static constexpr int kHalves = D / 64;
  static constexpr int kTile = kHalves * kHalf;
  static constexpr int kStages = D == 128 ? 5 : 8;  // K and V tiles in flight
  static constexpr int kKv = 2 * kTile;
  static constexpr int kBars = kKv + kStages * kTile;
  static constexpr int kNumBars = 2 * kStages + 2 + 2 + 2 + 2 + 1;
  static constexpr int kMisc = kBars + 8 * kNumBars;
  static constexpr int kTotal = kMisc + 16 + 1024;  // 1024: the tiles start on a swizzle atom
  static_assert(kTotal <= 227 * 1024, "shared memory");
};

// Tile t of the call -> its sequence.  Sequence b's tiles start at
// floor(off[b] / span) + b, which leaves room for its ceil(length / span) tiles
// without a sum over the sequences before it; a few numbers stay unused.
__device__ __forceinline__ int tile_sequence(const TcArgs& a, int tile, int span) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = a.sequences;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, b = lo + lane * step;
    const bool before = b < hi && clamp_to(a.q_off[b], a.total_q) / span + b <= tile;
    const int n = __popc(__ballot_sync(0xffffffffu, before));
    if (n == 0) return -1;
    lo += (n - 1) * step;
    hi = min(hi, lo + step);
    if (step == 1) break;
  }
  return lo;
}

// One CTA: two tiles of 128 query rows (tokens x the heads that share a KV
// head) against the keys of their sequence, 128 keys a step:
//   warp 9   copies Q, then K and V tiles through a ring (TMA);
//   warp 8   issues S = Q K^T into TMEM and O += P V with P from TMEM
//            (tcgen05.mma; tile 0's and tile 1's in turn, so that the tensor
//            core works on one tile while the other's softmax runs);
//   warps 0-3 and 4-7, one thread per row: running maximum, p = 2^(s - m),
//            P in 16 bits over S's columns, row sums in 32 bits.
// The row maximum that the exponents subtract only moves when it rises by more
// than 2^kSlack, so O (in TMEM) is rescaled rarely; S of step i + 1 is issued
// after P V of step i, so a completed S also says that O is at rest.
template <int D, bool BF16>
__global__ void __launch_bounds__(320, 1) attention_tc_kernel(const TcArgs a, const __grid_constant__ TcMaps maps) {
  using L = TcLayout<D>;
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  extern __shared__ uint8_t sm_raw[];
  uint8_t* sm = sm_raw + ((1024 - (ptx::saddr(sm_raw) & 1023)) & 1023);
  const unsigned sbase = ptx::saddr(sm);
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(sm + L::kBars);
  uint64_t* kv_empty = kv_full + L::kStages;
  uint64_t* q_full = kv_empty + L::kStages;  // [2] per tile
  uint64_t* s_full = q_full + 2;             // [2] scores complete (and the O before them)
  uint64_t* p_full = s_full + 2;             // [2] probabilities stored
  uint64_t* o_full = p_full + 2;             // [2] output complete
  uint64_t* drained = o_full + 2;
  unsigned* tmem_slot = reinterpret_cast<unsigned*>(sm + L::kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + L::kMisc + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // ---- which rows and keys ----
  const int kvh = blockIdx.x % a.kv_heads;
  const int split = (blockIdx.x / a.kv_heads) % a.splits;
  const int tile = a.tiles - 1 - blockIdx.x / (a.kv_heads * a.splits);  // causal: long tiles first
  const int span = 2 * a.tokens;
  ptx::griddep_launch();
  int seq = 0, q0 = 0, q_len = (int)a.total_q, k0 = 0, k_len = (int)a.total_k, first = 0;
  if (a.q_off) {
    seq = tile_sequence(a, tile, span);
    if (seq < 0) return;
    q0 = clamp_to(a.q_off[seq], a.total_q);
    q_len = clamp_to(a.q_off[seq + 1], a.total_q) - q0;
    k0 = clamp_to(a.k_off[seq], a.total_k);
    k_len = max(0, clamp_to(a.k_off[seq + 1], a.total_k) - k0);
    first = q0 / span + seq;
  }
  const int tok0 = (tile - first) * span;  // first token of the pair within the sequence
  if (tok0 < 0 || tok0 >= q_len) return;
  int end[2];  // keys that some row of the tile sees
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const int t_end = min(tok0 + (w + 1) * a.tokens, q_len);
    const bool any = tok0 + w * a.tokens < q_len;
    end[w] = !any ? 0 : a.causal ? max(0, min(k_len, t_end + k_len - q_len)) : k_len;
  }
  const int steps_all = (max(end[0], end[1]) + kKeys - 1) / kKeys;
  const int ja = (int)((long long)steps_all * split / a.splits), jb = (int)((long long)steps_all * (split + 1) / a.splits);
  const int cnt0 = max(0, min(jb, (end[0] + kKeys - 1) / kKeys) - ja);
  const int cnt1 = max(0, min(jb, (end[1] + kKeys - 1) / kKeys) - ja);
  const int cnt = max(cnt0, cnt1);

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::kStages; ++s) {
      ptx::mbar_init(&kv_full[s], 1);
      ptx::mbar_init(&kv_empty[s], 1);
    }
    for (int w = 0; w < 2; ++w) {
      ptx::mbar_init(&q_full[w], 1);
      ptx::mbar_init(&s_full[w], 1);
      ptx::mbar_init(&p_full[w], 4);
      ptx::mbar_init(&o_full[w], 1);
    }
    ptx::mbar_init(drained, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(ptx::saddr(tmem_slot))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const unsigned tmem = *tmem_slot;  // columns: S0 0, S1 128, O0 256, O1 256 + D

  if (warp == 9) {
    // ---- copies: ring slot of K step i: 2i, of V step i: 2i + 1 ----
    if (lane == 0) {
      int n = 0;  // ring tiles issued
      bool ok = true;
      auto load_kv = [&](const CUtensorMap* map, int i) {
        const int st = n % L::kStages;
        if (n >= L::kStages)
          ok = ok && ptx::wait_phase(&kv_empty[st], (n / L::kStages - 1) & 1, abort_flag, a.err, kAttnWaitFree);
        if (!ok) return;
        ptx::mbar_expect_tx(&kv_full[st], L::kTile);
        for (int h = 0; h < L::kHalves; ++h)
          ptx::tma_load_3d(sbase + L::kKv + st * L::kTile + h * L::kHalf, map, h * 64, kvh, k0 + (ja + i) * kKeys,
                           &kv_full[st]);
        ++n;
      };
      auto load_q = [&](int w) {
        if ((w == 0 ? cnt0 : cnt1) == 0) return;
        ptx::mbar_expect_tx(&q_full[w], (unsigned)(a.tokens * a.group * 128 * L::kHalves));
        for (int h = 0; h < L::kHalves; ++h)
          ptx::tma_load_4d(sbase + w * L::kTile + h * L::kHalf, &maps.q, h * 64, 0, kvh, q0 + tok0 + w * a.tokens,
                           &q_full[w]);
      };
      load_q(0);
      if (cnt > 0) load_kv(&maps.k, 0);
      load_q(1);
      for (int i = 0; i < cnt && ok; ++i) {
        load_kv(&maps.v, i);
        if (i + 1 < cnt && ok) load_kv(&maps.k, i + 1);
      }
      // Copies in flight land before the CTA exits.
      for (int s = max(0, n - L::kStages); s < n; ++s)
        ptx::wait_phase(&kv_full[s % L::kStages], (s / L::kStages) & 1, abort_flag, a.err, kAttnWaitLoad, false);
      if (cnt0 > 0) ptx::wait_phase(&q_full[0], 0, abort_flag, a.err, kAttnWaitLoad, false);
      if (cnt1 > 0) ptx::wait_phase(&q_full[1], 0, abort_flag, a.err, kAttnWaitLoad, false);
    }
    __syncwarp();
  } else if (warp == 8) {
    // ---- MMAs ----
    const unsigned id_s = ptx::idesc_f16(BF16, false, kRows, kKeys);
    const int n_o = (a.head_size + 15) / 16 * 16;  // channels past head_size are zeros (TMA fill)
    const unsigned id_o = ptx::idesc_f16(BF16, true, kRows, n_o);
    const int k_s = n_o / 16;
    bool ok = true;
    auto wait = [&](uint64_t* bar, unsigned parity, int code) {
      ok = ok && __all_sync(0xffffffffu, ptx::wait_phase(bar, parity, abort_flag, a.err, code));
      ptx::tc_fence_after();
    };
    auto ring = [&](int n) { return sbase + L::kKv + (n % L::kStages) * L::kTile; };
    auto ring_wait = [&](int n) { wait(&kv_full[n % L::kStages], (n / L::kStages) & 1, kAttnWaitLoad); };
    auto scores = [&](int w, int i) {  // S_w = Q_w K_i^T
      if (lane == 0) {
        const unsigned q = sbase + w * L::kTile, k = ring(2 * i);
        for (int s = 0; s < k_s; ++s) {
          const unsigned off = (s >> 2) * L::kHalf + (s & 3) * 32;
          ptx::tc_mma_ss(tmem + w * kKeys, ptx::smem_desc_128b(q + off, 16, 1024), ptx::smem_desc_128b(k + off, 16, 1024),
                         id_s, s > 0);
        }
        ptx::tc_commit(&s_full[w]);
      }
      __syncwarp();
    };
    if (cnt > 0) ring_wait(0);
    for (int w = 0; w < 2 && ok; ++w)
      if ((w ? cnt1 : cnt0) > 0) {
        wait(&q_full[w], 0, kAttnWaitLoad);
        if (ok) scores(w, 0);
      }
    if (ok && cnt > 0 && lane == 0) ptx::tc_commit(&kv_empty[0]);
    __syncwarp();
    for (int i = 0; i < cnt && ok; ++i) {
      ring_wait(2 * i + 1);
      if (!ok) break;
      // Value rows behind the last key that a row sees are not the sequence's
      // own, or masked for every row here: 0 x what they hold must stay 0.
      const int most = min(max(end[0], end[1]) - (ja + i) * kKeys, kKeys), padded = (most + 15) / 16 * 16;
      if (most < padded) {
        uint8_t* v = sm + L::kKv + ((2 * i + 1) % L::kStages) * L::kTile;
        for (int c = lane; c < (padded - most) * 8; c += 32)
          for (int h = 0; h < L::kHalves; ++h)
            *reinterpret_cast<uint4*>(v + h * L::kHalf + (most + c / 8) * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      }
      bool have_k = false;
      for (int w = 0; w < 2 && ok; ++w) {
        const int mine = w ? cnt1 : cnt0;
        if (i >= mine) continue;
        wait(&p_full[w], i & 1, kAttnWaitSoftmax);
        if (!ok) break;
        if (lane == 0) {
          const unsigned v = ring(2 * i + 1);
          const int steps = (min(end[w] - (ja + i) * kKeys, kKeys) + 15) / 16;
          for (int s = 0; s < steps; ++s)
            ptx::tc_mma_ts(tmem + 256 + w * D, tmem + w * kKeys + s * 8,
                           ptx::smem_desc_128b(v + s * 2048, L::kHalf, 1024), id_o, i > 0 || s > 0);
        }
        __syncwarp();
        if (i + 1 < mine) {
          if (!have_k) ring_wait(2 * i + 2);
          have_k = true;
          if (ok) scores(w, i + 1);
        } else if (lane == 0) {
          ptx::tc_commit(&o_full[w]);
        }
        __syncwarp();
      }
      if (ok && lane == 0) {
        ptx::tc_commit(&kv_empty[(2 * i + 1) % L::kStages]);
        if (i + 1 < cnt) ptx::tc_commit(&kv_empty[(2 * i + 2) % L::kStages]);
      }
      __syncwarp();
    }
    if (lane == 0 && !ok) {  // MMAs in flight finish before their memory is freed
      ptx::tc_commit(drained);
      ptx::wait_phase(drained, 0, abort_flag, a.err, kAttnWaitMma, false);
    }
    __syncwarp();
  } else {
    // ---- softmax: thread = query row ----
    const int w = warp >> 2;
    const int r = threadIdx.x & 127;
    const unsigned lanes = (unsigned)(32 * (warp & 3)) << 16;
    const unsigned s_addr = tmem + lanes + w * kKeys, o_addr = tmem + lanes + 256 + w * D;
    const int tok_in = r / a.group, g = r - tok_in * a.group;
    const int tok = tok0 + w * a.tokens + tok_in;
    const bool live = tok_in < a.tokens && tok < q_len;
    const int sees = !live ? 0 : a.causal ? max(0, min(k_len, tok + k_len - q_len + 1)) : k_len;
    const int mine = w ? cnt1 : cnt0;
    const float c = a.scale_log2;
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int i = 0; i < mine; ++i) {
      ok = __all_sync(0xffffffffu, ptx::wait_phase(&s_full[w], i & 1, abort_flag, a.err, kAttnWaitMma));
      if (!ok) break;
      ptx::tc_fence_after();
      unsigned u[128];
      float* s = reinterpret_cast<float*>(u);
#pragma unroll
      for (int k = 0; k < 4; ++k) ptx::tmem_ld32(s_addr + 32 * k, u + 32 * k);
      ptx::tc_wait_ld();
      const int lim = sees - (ja + i) * kKeys;
      if (__any_sync(0xffffffffu, lim < kKeys)) {
#pragma unroll
        for (int k = 0; k < kKeys; ++k)
          if (k >= lim) s[k] = -INFINITY;
      }
      float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int k = 4; k < kKeys; ++k) top[k & 3] = fmaxf(top[k & 3], s[k]);
      const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      if (i == 0) {
        m = mx;
      } else {
        const bool rise = mx * c > m * c + kSlack;
        if (__any_sync(0xffffffffu, rise)) {
          const float f = rise ? ptx::ex2((m - mx) * c) : 1.0f;
          if (rise) m = mx;
          l *= f;
#pragma unroll 1
          for (int k = 0; k < D; k += 32) {
            unsigned o[32];
            ptx::tmem_ld32(o_addr + k, o);
            ptx::tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            ptx::tmem_st32(o_addr + k, o);
          }
        }
      }
      const float base = m == -INFINITY ? 0.0f : m * c;
      float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        unsigned p[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float p0 = ptx::ex2(fmaf(s[32 * k + 2 * e], c, -base));
          const float p1 = ptx::ex2(fmaf(s[32 * k + 2 * e + 1], c, -base));
          sum[(2 * e) & 3] += p0;
          sum[(2 * e + 1) & 3] += p1;
          p[e] = ptx::pack16<BF16>(p0, p1);
        }
        ptx::tmem_st16(s_addr + 16 * k, p);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      ptx::tc_wait_st();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&p_full[w]);
    }
    if (ok && mine > 0) ok = __all_sync(0xffffffffu, ptx::wait_phase(&o_full[w], 0, abort_flag, a.err, kAttnWaitMma));
    if (ok) {
      ptx::tc_fence_after();
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const long long t = q0 + tok;
      const int h = kvh * a.group + g;
      const long long row = t * a.heads + h;
      T* out = static_cast<T*>(a.out) + t * a.out_token + h * a.out_head;
      float* part = a.part_o + (split * a.total_q * a.heads + row) * a.head_size;
#pragma unroll 1
      for (int k = 0; k < a.head_size; k += 32) {
        unsigned o[32];
        if (mine > 0) {
          ptx::tmem_ld32(o_addr + k, o);
          ptx::tc_wait_ld();
        }
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = l == 0.0f ? 0.0f : __uint_as_float(o[e]) * inv;
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          if (!live || k + e >= a.head_size) continue;
          if (a.splits > 1) {
            *reinterpret_cast<float4*>(part + k + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
            *reinterpret_cast<float4*>(part + k + e + 4) = make_float4(v[e + 4], v[e + 5], v[e + 6], v[e + 7]);
          } else {
            *reinterpret_cast<uint4*>(out + k + e) =
                make_uint4(ptx::pack16<BF16>(v[e], v[e + 1]), ptx::pack16<BF16>(v[e + 2], v[e + 3]),
                           ptx::pack16<BF16>(v[e + 4], v[e + 5]), ptx::pack16<BF16>(v[e + 6], v[e + 7]));
          }
        }
      }
      const float lse = (m == -INFINITY ? 0.0f : m * a.scale) + logf(l);
      if (live && a.splits > 1) a.part_lse[split * a.total_q * a.heads + row] = lse;
      if (live && a.splits == 1 && a.lse) a.lse[row] = lse;
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    ptx::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// Joins the parts of a row: lse = log sum_s e^lse_s, out = sum_s e^(lse_s - lse) o_s,
// in the order of the splits.  One warp per row.
template <typename T>
__global__ void __launch_bounds__(128) join_kernel(const TcArgs a) {
  const long long rows = a.total_q * a.heads, row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  ptx::griddep_wait();
  if (row >= rows) return;
  const long long t = row / a.heads;
  const int h = (int)(row - t * a.heads);
  if (a.q_off && (t < a.q_off[0] || t >= a.q_off[a.sequences])) return;
  float top = -INFINITY;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, a.part_lse[s * rows + row]);
  const float base = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f, o[4] = {};
  const int c = lane * 4;
  for (int s = 0; s < a.splits; ++s) {
    const float f = expf(a.part_lse[s * rows + row] - base);
    sum += f;
    if (c < a.head_size) {
      const float4 v = *reinterpret_cast<const float4*>(a.part_o + (s * rows + row) * a.head_size + c);
      o[0] = fmaf(f, v.x, o[0]);
      o[1] = fmaf(f, v.y, o[1]);
      o[2] = fmaf(f, v.z, o[2]);
      o[3] = fmaf(f, v.w, o[3]);
    }
  }
  if (c < a.head_size) {
    T* out = static_cast<T*>(a.out) + t * a.out_token + h * a.out_head;
    T v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (T)(sum == 0.0f ? 0.0f : o[i] / sum);
    *reinterpret_cast<uint2*>(out + c) = *reinterpret_cast<const uint2*>(v);
  }
  if (a.lse && lane == 0) a.lse[row] = base + logf(sum);
}

// ------------------------------------------------------------- launch ----

// Byte stride of a tensor map dimension; one of length 1 has none to speak of.
cuuint64_t map_stride(int64_t extent, int64_t stride) { return extent == 1 ? 16 : (cuuint64_t)stride * 2; }

CUtensorMapDataType map_type(int dtype) {
  return dtype == FA_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

// K or V: (channel, KV head, key), 64 channels x 128 keys a copy.
void encode_kv(CUtensorMap* m, int dtype, const void* base, int head_size, int kv_heads, int64_t keys, const int64_t* stride) {
  const cuuint64_t dims[3] = {(cuuint64_t)head_size, (cuuint64_t)kv_heads, (cuuint64_t)keys};
  const cuuint64_t strides[2] = {map_stride(kv_heads, stride[1]), map_stride(keys, stride[0])};
  const cuuint32_t box[3] = {64, 1, kKeys};
  encode_tensor_map(m, map_type(dtype), 3, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int D, bool BF16>
void launch_tc(const TcArgs& t, const TcMaps& maps, cudaStream_t stream) {
  FA_CUDA(cudaFuncSetAttribute(attention_tc_kernel<D, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               TcLayout<D>::kTotal));
  const unsigned grid = (unsigned)t.tiles * t.kv_heads * t.splits;
  attention_tc_kernel<D, BF16><<<grid, 320, TcLayout<D>::kTotal, stream>>>(t, maps);
  FA_CUDA(cudaGetLastError());
}

int* error_word() {
  void* p = nullptr;
  FA_CUDA(cudaGetSymbolAddress(&p, g_dev_error));
  return static_cast<int*>(p);
}

// Tile pairs of a packed call, an upper bound (tile_sequence).
int64_t tile_pairs(int64_t total_q, int sequences, int group) { return total_q / (2 * (kRows / group)) + sequences; }

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
  TcArgs t;
  t.q_off = a.q_offsets;
  t.k_off = a.k_offsets;
  t.sequences = a.sequences;
  t.total_q = a.total_q;
  t.total_k = a.total_k;
  t.heads = a.heads;
  t.kv_heads = a.kv_heads;
  t.group = a.heads / a.kv_heads;
  t.head_size = a.head_size;
  t.tokens = kRows / t.group;
  t.tiles = (int)tile_pairs(a.total_q, a.sequences, t.group);
  t.causal = a.causal;
  t.scale = a.scale;
  t.scale_log2 = (float)(a.scale * 1.4426950408889634);
  t.out = a.out;
  t.out_token = a.out_stride[0];
  t.out_head = a.out_stride[1];
  t.lse = a.lse;
  t.err = error_word();
  TcMaps maps;
  {
    const cuuint64_t dims[4] = {(cuuint64_t)a.head_size, (cuuint64_t)t.group, (cuuint64_t)a.kv_heads,
                                (cuuint64_t)a.total_q};
    const cuuint64_t strides[3] = {map_stride(t.group, a.q_stride[1]),
                                   map_stride(a.kv_heads, a.q_stride[1] * t.group), map_stride(a.total_q, a.q_stride[0])};
    const cuuint32_t box[4] = {64, (cuuint32_t)t.group, 1, (cuuint32_t)t.tokens};
    encode_tensor_map(&maps.q, map_type(a.dtype), 4, a.q, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  }
  if (a.total_k > 0) {
    encode_kv(&maps.k, a.dtype, a.k, a.head_size, a.kv_heads, a.total_k, a.k_stride);
    encode_kv(&maps.v, a.dtype, a.v, a.head_size, a.kv_heads, a.total_k, a.v_stride);
  } else {
    maps.k = maps.v = maps.q;  // never used: no sequence has a key
  }
  const bool bf16 = a.dtype == FA_DTYPE_BF16;
  if (a.head_size <= 64)
    bf16 ? launch_tc<64, true>(t, maps, stream) : launch_tc<64, false>(t, maps, stream);
  else
    bf16 ? launch_tc<128, true>(t, maps, stream) : launch_tc<128, false>(t, maps, stream);
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
