// Attention over packed sequences and over a shared prefix (fa_dev_attention_*).
//
//     out_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_i . k_j - m_i)
//
// over the keys j that query i sees, in one pass with the running maximum m_i.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <map>
#include <mutex>
#include <vector>

#include "dev_ops.h"
#include "dev_ptx.cuh"
#include "tma_host.h"

namespace fa {

namespace {

// A word per backend.  Module memory, so that a captured graph may outlive the
// backend whose word it would set; backends beyond kErrorWords share words.
constexpr int kErrorWords = 4096;
__device__ int g_dev_errors[kErrorWords];
std::mutex g_words_mu;
std::map<int, std::vector<int>> g_word_users;  // by device

// ------------------------------------------------------------- checks ----

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

void need(bool ok, const char* what) {
  if (!ok) throw Error(kErrArgument, what);
}

// Strides in elements of two bytes: every row must start on 16 bytes (a
// dimension of length one has a single start).
bool strides16(const int64_t* s, std::initializer_list<int64_t> extents) {
  for (int64_t n : extents)
    if (*s++ % 8 != 0 && n > 1) return false;
  return true;
}

void need_strides(const int64_t* s, int n) {
  for (int i = 0; i < n; ++i) need(s[i] >= 0 && s[i] < (1ll << 38), "a stride is negative or beyond 2^38 elements");
}

// Whether no two elements of a strided output share a place (strides as need_strides leaves them).
bool apart(const int64_t* strides, const int64_t* extents, int64_t inner) {
  int order[2] = {0, 1};
  if (strides[1] < strides[0]) std::swap(order[0], order[1]);
  int64_t span = inner;
  for (int d : order) {
    if (extents[d] <= 1) continue;
    if (strides[d] < span) return false;
    span = (int64_t)std::min((double)span + (double)strides[d] * (double)(extents[d] - 1), 1e12);  // beyond any stride
  }
  return true;
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

__device__ __forceinline__ int clamp_to(int x, long long hi) { return (int)min((long long)max(x, 0), hi); }

// -------------------------------------------------- tensor-core attention ----

constexpr int kRows = 128;     // query rows of one tile (TMEM lanes): tokens x heads of a KV head's group
constexpr int kKeys = 128;     // keys of a K or V tile in shared memory
constexpr int kUnit = 64;      // keys per softmax step: half a tile
constexpr float kSlack = 8.0f; // powers of two by which a row's maximum may rise before its sums are rescaled

enum AttnError : int {
  kAttnWaitLoad = 41,
  kAttnWaitMma = 42,
  kAttnWaitSoftmax = 43,
  kAttnWaitFree = 44,
  kAttnWaitTest = 45
};

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
  float* part_o = nullptr;     // with part_o: [splits x total_q x heads x head_size], and the rows' lse
  float* part_lse = nullptr;
  int* err = nullptr;
  // What the maps describe, for rows that a masked value spoiled (mend_rows).
  const void *q = nullptr, *k = nullptr, *v = nullptr;
  long long q_token = 0, q_head = 0, k_token = 0, k_head = 0, v_token = 0, v_head = 0;
};
struct TcMaps {
  CUtensorMap q;  // (channel, head of the group, KV head, token)
  CUtensorMap k;  // (channel, KV head, key)
  CUtensorMap v;
};

// W tiles of kRows query rows per CTA.
template <int D, int W>
struct TcLayout {
  static constexpr int kThreads = W * 160 + 32;     // per tile 4 softmax warps and 1 that issues MMAs; 1 that copies
  // A tile of Q: 128 rows in halves of 64 channels with 128-byte swizzle; of K
  // and V: kTileKeys rows alike.
  static constexpr int kHalves = D / 64, kQHalf = kRows * 128, kQ = kHalves * kQHalf;
  static constexpr int kTileKeys = W == 2 ? 128 : kUnit;
  static constexpr int kHalf = kTileKeys * 128, kTile = kHalves * kHalf;
  static constexpr int kStages = D == 128 ? 5 : 8;  // K and V tiles in flight
  static constexpr int kKv = W * kQ;
  static constexpr int kBars = kKv + kStages * kTile;
  static constexpr int kNumBars = 2 * kStages + 2 + 4 + 4 + 4 + 2;
  static constexpr int kMisc = (kBars + 8 * kNumBars + 15) / 16 * 16;
  static constexpr int kWork = kMisc + 16;  // the CTA's Work
  static constexpr int kTotal = kWork + 64;
  // TMEM columns: tile w's S buffers at 128 w and 128 w + 64, its O at kO + w D.
  static constexpr int kO = W * 128, kColumns = W * 256;
  static_assert(kO + W * D <= kColumns, "TMEM");
  static_assert(kTotal <= (W == 2 ? 227 : 113) * 1024, "shared memory of one or two CTAs an SM");
};

// What a CTA does, worked out by its last warp: place (below), then keys.
struct __align__(16) Work {
  int q0, q_len, k0, k_len, tok0;  // tok0 < 0: nothing
  int end[2];                      // keys that some row of the tile sees
  int key0, key1;                  // this split's keys: first, and behind the last
  int cnt[2];                      // steps of the tiles
  int ring;                        // copies of K and V
};

// Where a CTA works: its sequence's queries and keys, and its first query token.
struct Place {
  int q0 = 0, q_len = 0, k0 = 0, k_len = 0, token = -1;  // token < 0: nowhere
};

// Number t of the call -> its place, for up to 32 sequences: a lane per sequence.
// Sequences with more keys come first, and in each the last tile first (it sees
// the most keys): the SMs that finish early take the short ones (in their own
// order: frames both ways 78 us instead of 68, chunks on a history 143, not 102).
__device__ __forceinline__ Place place_sorted(const TcArgs& a, int t, int span) {
  const int lane = threadIdx.x & 31;
  Place p;
  if (lane < a.sequences) {
    p.q0 = clamp_to(a.q_off[lane], a.total_q);
    p.q_len = clamp_to(a.q_off[lane + 1], a.total_q) - p.q0;
    p.k0 = clamp_to(a.k_off[lane], a.total_k);
    p.k_len = max(0, clamp_to(a.k_off[lane + 1], a.total_k) - p.k0);
  }
  const int mine = p.q_len > 0 ? (p.q_len + span - 1) / span : 0;
  int start = 0;  // tiles of the sequences before this lane's
  for (int j = 0; j < a.sequences; ++j) {
    const int k = __shfl_sync(0xffffffffu, p.k_len, j), n = __shfl_sync(0xffffffffu, mine, j);
    if (k > p.k_len || (k == p.k_len && j < lane)) start += n;
  }
  const unsigned here = __ballot_sync(0xffffffffu, t >= start && t < start + mine);
  if (here == 0) return Place{};
  const int b = __ffs(here) - 1;
  p.token = (mine - 1 - (t - start)) * span;
  p.q0 = __shfl_sync(0xffffffffu, p.q0, b);
  p.q_len = __shfl_sync(0xffffffffu, p.q_len, b);
  p.k0 = __shfl_sync(0xffffffffu, p.k0, b);
  p.k_len = __shfl_sync(0xffffffffu, p.k_len, b);
  p.token = __shfl_sync(0xffffffffu, p.token, b);
  return p;
}

// The same for any number of sequences, in their own order from the last tile
// on.  Sequence b's tiles start at floor(off[b] / span) + b, which leaves room
// for its ceil(length / span) tiles without a sum over the sequences before it;
// a few numbers stay unused.
__device__ __forceinline__ Place place_searched(const TcArgs& a, int t, int span) {
  const int lane = threadIdx.x & 31, tile = a.tiles - 1 - t;
  int lo = 0, hi = a.sequences;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, b = lo + lane * step;
    const bool before = b < hi && clamp_to(a.q_off[b], a.total_q) / span + b <= tile;
    const int n = __popc(__ballot_sync(0xffffffffu, before));
    if (n == 0) return Place{};
    lo += (n - 1) * step;
    hi = min(hi, lo + step);
    if (step == 1) break;
  }
  Place p;
  p.q0 = clamp_to(a.q_off[lo], a.total_q);
  p.q_len = clamp_to(a.q_off[lo + 1], a.total_q) - p.q0;
  p.k0 = clamp_to(a.k_off[lo], a.total_k);
  p.k_len = max(0, clamp_to(a.k_off[lo + 1], a.total_k) - p.k0);
  const int i = tile - (p.q0 / span + lo);
  p.token = i >= 0 && i * (long long)span < p.q_len ? i * span : -1;
  return p;
}

__device__ __forceinline__ uint4 lds16(unsigned addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

// A masked key's probability is 0, but 0 x infinity and 0 x NaN are NaN: where a
// value behind the keys that a row sees (in the tile at the causal border) is
// not finite, the row is computed again without it.  All lanes of a warp, for
// the rows in `bad`: row r's lane has what it sees, its maximum (times the
// scale's log2), 1 / sum, its query and its head.  The result goes to the row's
// place in the stage, 4 channels a lane, from channel `from` on.
template <typename T>
__device__ __noinline__ void mend_rows(const TcArgs& a, unsigned bad, int first_key, int end_key, int sees, float base,
                                       float inv, long long token, int head, long long k0, int kvh, int from, int width,
                                       unsigned stage, int row_bytes) {
  const int lane = threadIdx.x & 31, c = from + lane * 4;
  const bool on = lane * 4 < width && c < a.head_size;
  auto load = [](const T* p, float* x) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)reinterpret_cast<const T*>(&u)[i];
  };
#pragma unroll 1
  for (; bad; bad &= bad - 1) {
    const int r = __ffs(bad) - 1;
    const int seen = min(__shfl_sync(0xffffffffu, sees, r), end_key);
    const float m = __shfl_sync(0xffffffffu, base, r), by = __shfl_sync(0xffffffffu, inv, r);
    const long long tok = __shfl_sync(0xffffffffu, token, r);
    const int h = __shfl_sync(0xffffffffu, head, r);
    const T* k = static_cast<const T*>(a.k) + k0 * a.k_token + kvh * a.k_head;
    const T* v = static_cast<const T*>(a.v) + k0 * a.v_token + kvh * a.v_head;
    bool spoiled = false;
#pragma unroll 1
    for (int j = max(seen, first_key); j < end_key; ++j) {
      float x[4] = {};
      if (on) load(v + j * a.v_token + c, x);
      spoiled |= !(isfinite(x[0]) && isfinite(x[1]) && isfinite(x[2]) && isfinite(x[3]));
    }
    if (!__any_sync(0xffffffffu, spoiled)) continue;  // what it sees is not finite
    const T* q = static_cast<const T*>(a.q) + tok * a.q_token + h * a.q_head;
    float o[4] = {}, qx[4] = {};
    const int cq = lane * 4;
    if (cq < a.head_size) load(q + cq, qx);
#pragma unroll 1
    for (int j = first_key; j < seen; ++j) {
      float kx[4] = {}, vx[4] = {}, dot = 0.0f;
      if (cq < a.head_size) load(k + j * a.k_token + cq, kx);
      if (on) load(v + j * a.v_token + c, vx);
#pragma unroll
      for (int i = 0; i < 4; ++i) dot = fmaf(qx[i], kx[i], dot);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
      const float p = ptx::ex2(fmaf(dot, a.scale_log2, -m));
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = fmaf(p, vx[i], o[i]);
    }
    if (lane * 4 >= width) continue;
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] *= by;
    const bool parts = a.part_o != nullptr;
    const int chunk = parts ? lane : lane / 2;
    const unsigned at = stage + r * row_bytes + ((chunk ^ (r & 7)) << 4) + (parts ? 0 : (lane & 1) * 8);
    if (parts)
      asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(o[0]), "f"(o[1]), "f"(o[2]), "f"(o[3]) : "memory");
    else
      asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(ptx::pack16<kBf16>(o[0], o[1])),
                   "r"(ptx::pack16<kBf16>(o[2], o[3]))
                   : "memory");
  }
}

// One CTA: W tiles of 128 query rows (tokens x the heads that share a KV head)
// against the keys of their sequence, 64 keys a step:
//   the last warp copies Q, then K and V tiles through a ring (TMA);
//   one warp per tile issues S = Q K^T into TMEM and O += P V with P from TMEM
//     (tcgen05.mma; one thread issues an MMA per ~62 cycles, an MMA of 64 keys
//     lasts 32 to 48: one issuer for both tiles was the bound);
//   four warps per tile, one thread per row: running maximum, p = 2^(s - m),
//     P in 16 bits over S's columns, row sums in 32 bits.
// W = 2: K and V tiles are read once for 256 rows.  W = 1: two CTAs share an SM,
// so that one's start and end (its first copies, its last rows' way out) pass
// while the other computes; for sequences of few steps.
// TMEM holds two S buffers of 64 keys per tile next to the two O: while a tile's
// softmax works on one buffer, the tensor core turns the other's P into O and
// refills it, so neither waits for the other's whole step.  The row maximum that
// the exponents subtract only moves when it rises by more than 2^kSlack, so O (in
// TMEM) is rescaled rarely (at every rise: long prompts 783 us instead of 500, a
// shared prefix for 256 sessions 158 instead of 108).  P is rounded to the type of
// V for the product with it, up to 2^kSlack, exactly as far as a P below 1 is;
// the sum of a row takes the values before that rounding.
//
// Bound: for D = 128 the MMAs and the shared memory that feeds them (with N = 64
// keys an S = Q K^T reads Q again for every 64 keys; the long prompts below
// took 526 and 498 us in two steps on the way, 510 without any exponential); for D = 64
// MMAs and exponentials alike, as many of the latter per key with half the products.  Two prompts of 8192 tokens, 16 query and 8 KV
// heads, bf16: 500 us, 1100 TFLOP/s of the 1689 that a library product reaches; 24
// prompts of 1 to 700 tokens: 50 us, where the starts and ends of the CTAs count.
template <int D, int W, bool BF16>
__global__ void __launch_bounds__((TcLayout<D, W>::kThreads), W == 2 ? 1 : 2)
    attention_tc_kernel(const __grid_constant__ TcArgs a, const __grid_constant__ TcMaps maps) {
  using L = TcLayout<D, W>;
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  extern __shared__ __align__(1024) uint8_t sm[];  // the tiles start on a swizzle atom
  const unsigned sbase = ptx::saddr(sm);
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(sm + L::kBars);
  uint64_t* kv_empty = kv_full + L::kStages;
  uint64_t* q_full = kv_empty + L::kStages;  // [2] per tile
  uint64_t* s_full = q_full + 2;             // [2 tiles x 2 buffers] scores complete
  uint64_t* p_full = s_full + 4;             // [2 x 2] probabilities stored
  uint64_t* pv_done = p_full + 4;            // [2 x 2] their product with V added to O
  uint64_t* drained = pv_done + 4;           // [2]
  unsigned* tmem_slot = reinterpret_cast<unsigned*>(sm + L::kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + L::kMisc + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // ---- which rows and keys ----
  if (warp == 5 * W && lane == 0) {
    ptx::prefetch_map(&maps.k);
    ptx::prefetch_map(&maps.q);
    ptx::prefetch_map(&maps.v);
    for (int s = 0; s < L::kStages; ++s) {
      ptx::mbar_init(&kv_full[s], 1);
      ptx::mbar_init(&kv_empty[s], W);  // every issuer
    }
    for (int w = 0; w < 2; ++w) {
      ptx::mbar_init(&q_full[w], 1);
      ptx::mbar_init(&drained[w], 1);
    }
    for (int b = 0; b < 4; ++b) {
      ptx::mbar_init(&s_full[b], 1);
      ptx::mbar_init(&p_full[b], 4);
      ptx::mbar_init(&pv_done[b], 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  const int kvh = blockIdx.x % a.kv_heads;
  int number = blockIdx.x / a.kv_heads, split = 0;
  if (a.splits > 1) {
    split = number % a.splits;
    number /= a.splits;
  }
  ptx::griddep_launch();

  // Ring number of K tile i: 2i, of V tile i: 2i + 1, for keys from `first` on.
  auto load_kv = [&](int n, int first) {
    const int st = n % L::kStages;
    ptx::mbar_expect_tx(&kv_full[st], L::kTile);
    for (int h = 0; h < L::kHalves; ++h)
      ptx::tma_load_3d(sbase + L::kKv + st * L::kTile + h * L::kHalf, n & 1 ? &maps.v : &maps.k, h * 64, kvh,
                       first + (n >> 1) * L::kTileKeys, &kv_full[st]);
  };
  // One warp works out the CTA's place and sends for the first tiles while the
  // others wait (their copies of that code only fought for the same units).
  Work* work = reinterpret_cast<Work*>(sm + L::kWork);
  if (warp == 5 * W) {
    const int span = W * a.tokens;
    Place at;
    if (a.q_off) {
      at = a.sequences <= 32 ? place_sorted(a, number, span) : place_searched(a, number, span);
    } else {
      at.q_len = (int)a.total_q;
      at.k_len = (int)a.total_k;
      at.token = number * span;
    }
    Work x;
    x.q0 = at.q0;
    x.q_len = at.q_len;
    x.k0 = at.k0;
    x.k_len = at.k_len;
    x.tok0 = at.token;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const int t_end = min(at.token + (w + 1) * a.tokens, at.q_len);
      const bool any = w < W && at.token >= 0 && at.token + w * a.tokens < at.q_len;
      x.end[w] = !any ? 0 : a.causal ? max(0, min(at.k_len, t_end + at.k_len - at.q_len)) : at.k_len;
    }
    const int tiles = (max(x.end[0], x.end[1]) + kKeys - 1) / kKeys;
    int ja = 0, jb = tiles;
    if (a.splits > 1) {  // as even as tiles allow: the first `over` splits have one more
      const int each = tiles / a.splits, over = tiles - each * a.splits;
      ja = split * each + min(split, over);
      jb = ja + each + (split < over);
    }
    x.key0 = ja * kKeys;
    x.key1 = jb * kKeys;
#pragma unroll
    for (int w = 0; w < 2; ++w) x.cnt[w] = max(0, (min(x.key1, x.end[w]) - x.key0 + kUnit - 1) / kUnit);
    x.ring = 2 * ((max(x.cnt[0], x.cnt[1]) * kUnit + L::kTileKeys - 1) / L::kTileKeys);
    if (lane == 0) {
      *work = x;
      if (x.ring > 0) load_kv(0, x.k0 + x.key0);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if (x.cnt[w] == 0) continue;
        ptx::mbar_expect_tx(&q_full[w], (unsigned)(a.tokens * a.group * 128 * L::kHalves));
        for (int h = 0; h < L::kHalves; ++h)
          ptx::tma_load_4d(sbase + w * L::kQ + h * L::kQHalf, &maps.q, h * 64, 0, kvh, x.q0 + x.tok0 + w * a.tokens,
                           &q_full[w]);
      }
    }
  }
  if (warp == 4 * W) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ptx::saddr(tmem_slot)),
                 "n"(L::kColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const int q0 = work->q0, q_len = work->q_len, k0 = work->k0, k_len = work->k_len, tok0 = work->tok0;
  const int end_all = max(work->end[0], work->end[1]), key0 = work->key0, key1 = work->key1;
  const int cnt0 = work->cnt[0], cnt1 = work->cnt[1], cnt = max(cnt0, cnt1), ring = work->ring;
  if (tok0 < 0) {
    if (warp == 4 * W) ptx::tmem_free<L::kColumns>(*tmem_slot);
    return;
  }
  // All 512 columns start at 0; half of them where the SM's other CTA is not.
  const unsigned tm = W == 2 ? 0 : __shfl_sync(0xffffffffu, *tmem_slot, 0);

  if (warp == 5 * W) {
    // ---- the other copies ----
    if (lane == 0) {
      int n = min(ring, 1);
#pragma unroll 1
      for (; n < ring; ++n) {
        if (n >= L::kStages && !ptx::wait_phase(&kv_empty[n % L::kStages], (n / L::kStages - 1) & 1, abort_flag, a.err, kAttnWaitFree)) break;
        load_kv(n, k0 + key0);
      }
      // Copies in flight land before the CTA exits.
#pragma unroll 1
      for (int s = max(0, n - L::kStages); s < n; ++s)
        ptx::wait_phase(&kv_full[s % L::kStages], (s / L::kStages) & 1, abort_flag, a.err, kAttnWaitLoad, false);
      if (cnt0 > 0) ptx::wait_phase(&q_full[0], 0, abort_flag, a.err, kAttnWaitLoad, false);
      if (cnt1 > 0) ptx::wait_phase(&q_full[1], 0, abort_flag, a.err, kAttnWaitLoad, false);
    }
    __syncwarp();
  } else if (warp >= 4 * W) {
    // ---- MMAs of one tile, by one thread: constant offsets and no arithmetic
    // between the MMAs of a step, no votes between the waits ----
    if (ptx::elect()) {
      const int w = W == 2 ? warp - 8 : 0, mine = w ? cnt1 : cnt0;
      const unsigned id_s = ptx::idesc_f16(BF16, false, kRows, kUnit);
      const int n_o = (a.head_size + 15) / 16 * 16;  // channels past head_size are zeros (TMA fill)
      const unsigned id_o = ptx::idesc_f16(BF16, true, kRows, n_o);
      const int k_s = n_o / 16;
      bool ok = true;
      auto wait = [&](uint64_t* bar, unsigned parity, int code) {
        ok = ok && ptx::wait_phase(bar, parity, abort_flag, a.err, code);
      };
      const unsigned q_low = ptx::smem_desc_low(sbase + w * L::kQ, 16), k_low = ptx::smem_desc_low(sbase + L::kKv, 16),
                     v_low = ptx::smem_desc_low(sbase + L::kKv, L::kHalf);
      struct Slot {  // a tile's place in the ring; K tiles have even numbers, V tiles odd ones
        int st;
        unsigned ph;
        __device__ __forceinline__ void next() {
          st += 2;
          if (st >= L::kStages) {
            st -= L::kStages;
            ph ^= 1;
          }
        }
      };
      Slot ks{0, 0}, vs{1, 0};
      constexpr int kPart = W == 2 ? kUnit * 128 : 0;  // bytes between the steps of a tile
      const unsigned s_at = tm + w * 128, o_at = tm + L::kO + w * D;
      auto scores = [&](int b) {  // S_w of the K tile (W = 2: of its half b) into buffer b
        const unsigned k = k_low + ks.st * (L::kTile >> 4) + b * (kPart >> 4);
        if (k_s == D / 16) {
#pragma unroll
          for (int s = 0; s < D / 16; ++s)
            ptx::tc_mma_ss(s_at + b * kUnit, q_low + (((s >> 2) * L::kQHalf + (s & 3) * 32) >> 4),
                           k + (((s >> 2) * L::kHalf + (s & 3) * 32) >> 4), id_s, s > 0);
        } else {
#pragma unroll 1
          for (int s = 0; s < k_s; ++s)
            ptx::tc_mma_ss(s_at + b * kUnit, q_low + (((s >> 2) * L::kQHalf + (s & 3) * 32) >> 4),
                           k + (((s >> 2) * L::kHalf + (s & 3) * 32) >> 4), id_s, s > 0);
        }
        ptx::tc_commit(&s_full[2 * w + b]);
      };
      auto values = [&](int b, int steps, bool acc) {  // O_w += P_w (buffer b) x the V tile (its half b)
        const unsigned v = v_low + vs.st * (L::kTile >> 4) + b * (kPart >> 4);
        ptx::tc_fence_after();
        if (steps == kUnit / 16) {
#pragma unroll
          for (int s = 0; s < kUnit / 16; ++s)
            ptx::tc_mma_ts(o_at, s_at + b * kUnit + s * 8, v + (s * 2048 >> 4), id_o, acc || s > 0);
        } else {
#pragma unroll 1
          for (int s = 0; s < steps; ++s)
            ptx::tc_mma_ts(o_at, s_at + b * kUnit + s * 8, v + (s * 2048 >> 4), id_o, acc || s > 0);
        }
        ptx::tc_commit(&pv_done[2 * w + b]);
      };
      auto release = [&](int st) {
        if (ok) ptx::tc_commit(&kv_empty[st]);
      };
      const int end = work->end[w];
      auto steps_of = [&](int n) { return (min(end - key0 - n * kUnit, kUnit) + 15) / 16; };
      if (cnt > 0) wait(&kv_full[0], 0, kAttnWaitLoad);
      if (mine > 0) wait(&q_full[w], 0, kAttnWaitLoad);
      if (W == 1) {  // a tile a step
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          if (!ok || b >= mine) continue;
          if (b == 1) wait(&kv_full[ks.st], ks.ph, kAttnWaitLoad);
          if (ok) scores(b);
          release(ks.st);
          ks.next();
        }
#pragma unroll 1
        for (int n0 = 0; n0 < mine && ok; n0 += 2)
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int n = n0 + b;
            if (!ok || n >= mine) continue;
            wait(&kv_full[vs.st], vs.ph, kAttnWaitLoad);
            wait(&p_full[b], (n0 >> 1) & 1, kAttnWaitSoftmax);
            if (!ok) continue;
            values(b, steps_of(n), n > 0);
            release(vs.st);
            vs.next();
            if (n + 2 >= mine) continue;
            wait(&kv_full[ks.st], ks.ph, kAttnWaitLoad);
            if (ok) scores(b);
            release(ks.st);
            ks.next();
          }
      } else {
        if (ok && mine > 0) scores(0);
        if (ok && mine > 1) scores(1);
        if (cnt > 0) release(0);
        ks.next();
#pragma unroll 1
        for (int n0 = 0; n0 < cnt && ok; n0 += 2) {  // one V tile, and the K tile after its own
          // Waits, and releases below, also for tiles that only the other issuer uses:
          // one that ran ahead would release a slot's next use.
          wait(&kv_full[vs.st], vs.ph, kAttnWaitLoad);
          if (!ok) break;
          if (n0 + 2 < cnt) wait(&kv_full[ks.st], ks.ph, kAttnWaitLoad);
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int n = n0 + b;
            if (!ok || n >= mine) continue;
            wait(&p_full[2 * w + b], (n0 >> 1) & 1, kAttnWaitSoftmax);
            if (!ok) continue;
            values(b, steps_of(n), n > 0);
            if (n + 2 < mine) scores(b);
          }
          release(vs.st);
          if (n0 + 2 < cnt) release(ks.st);
          vs.next();
          ks.next();
        }
      }
      if (!ok) {  // MMAs in flight finish before their memory is freed
        ptx::tc_commit(&drained[w]);
        ptx::wait_phase(&drained[w], 0, abort_flag, a.err, kAttnWaitMma, false);
      }
    }
    __syncwarp();
  } else {
    // ---- softmax: thread = query row ----
    const int w = warp >> 2;
    const int r = threadIdx.x & 127;
    const unsigned lanes = (unsigned)(32 * (warp & 3)) << 16;
    const unsigned o_addr = tm + lanes + L::kO + w * D;
    const int tok_in = r / a.group, g = r - tok_in * a.group;
    const int tok = tok0 + w * a.tokens + tok_in;
    const bool live = tok_in < a.tokens && tok < q_len;
    const int sees = !live ? 0 : a.causal ? max(0, min(k_len, tok + k_len - q_len + 1)) : k_len;
    const int mine = w ? cnt1 : cnt0;
    const float c = a.scale_log2;
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
#pragma unroll 1
    for (int n = 0; n < mine && ok; ++n) {
      ok = __all_sync(0xffffffffu,
                      ptx::wait_phase(&s_full[2 * w + (n & 1)], (n >> 1) & 1, abort_flag, a.err, kAttnWaitMma));
      if (!ok) break;
      ptx::tc_fence_after();
      const unsigned s_addr = tm + lanes + w * 128 + (n & 1) * kUnit;
      const int lim = sees - key0 - n * kUnit;  // keys of this step that the row sees
      bool done = false;
      if (n > 0 && __all_sync(0xffffffffu, lim >= kUnit)) {
        // Every key is seen, and the maximum so far most likely serves: the
        // exponentials start with the first scores instead of after the last,
        // and count only if no score is too far above the maximum (long prompts:
        // 501 us, 559 without).
        const uint64_t c2 = ptx::pair(c, c);
        const float nb = m == -INFINITY ? 0.0f : -m * c;
        const uint64_t nb2 = ptx::pair(nb, nb);
        unsigned p[32], u[2][32];
        uint64_t sum[2] = {0, 0};
        float top[2] = {-INFINITY, -INFINITY};
        ptx::tmem_ld32(s_addr, u[0]);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          ptx::tc_wait_ld();
          if (k < 1) ptx::tmem_ld32(s_addr + 32, u[1]);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float s0 = __uint_as_float(u[k][2 * e]), s1 = __uint_as_float(u[k][2 * e + 1]);
            top[e & 1] = ptx::max3(top[e & 1], s0, s1);
            float x0, x1;
            ptx::unpair(ptx::fma2(ptx::pair(s0, s1), c2, nb2), x0, x1);
            x0 = ptx::ex2(x0);
            x1 = ptx::ex2(x1);
            sum[e & 1] = ptx::add2(sum[e & 1], ptx::pair(x0, x1));
            p[16 * k + e] = ptx::pack16<BF16>(x0, x1);
          }
        }
        done = !__any_sync(0xffffffffu, fmaxf(top[0], top[1]) * c > m * c + kSlack);
        if (done) {
          ptx::tmem_st32(s_addr, p);
          float a0, a1;
          ptx::unpair(ptx::add2(sum[0], sum[1]), a0, a1);
          l += a0 + a1;
        }
      }
      if (!done) {
        // The first step, masked keys, or a maximum that may move: all scores first.
        unsigned u[64];
        ptx::tmem_ld32(s_addr, u);
        ptx::tmem_ld32(s_addr + 32, u + 32);
        ptx::tc_wait_ld();
        if (__any_sync(0xffffffffu, lim < kUnit)) {
#pragma unroll
          for (int e = 0; e < kUnit; ++e)
            if (e >= lim) u[e] = 0xff800000u;  // -inf
        }
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < kUnit; e += 2)
          top[(e >> 1) & 3] = ptx::max3(top[(e >> 1) & 3], __uint_as_float(u[e]), __uint_as_float(u[e + 1]));
        const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        if (n == 0) {
          m = mx;
        } else {
          const bool rise = mx * c > m * c + kSlack;
          if (__any_sync(0xffffffffu, rise)) {
            // O is at rest once the step before is in it.
            ok = __all_sync(0xffffffffu,
                            ptx::wait_phase(&pv_done[2 * w + ((n - 1) & 1)], ((n - 1) >> 1) & 1, abort_flag, a.err,
                                            kAttnWaitMma));  // a failed wait ends the loop at the next one
            ptx::tc_fence_after();
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
        float sum[2] = {0.0f, 0.0f};
        unsigned p[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float p0 = ptx::ex2(fmaf(__uint_as_float(u[2 * e]), c, -base));
          const float p1 = ptx::ex2(fmaf(__uint_as_float(u[2 * e + 1]), c, -base));
          sum[0] += p0;
          sum[1] += p1;
          p[e] = ptx::pack16<BF16>(p0, p1);
        }
        ptx::tmem_st32(s_addr, p);
        l += sum[0] + sum[1];
      }
      // Value rows behind the last key that a row sees are not the sequence's own,
      // or masked for every row here: 0 x what they hold must stay 0.  The step
      // that takes some of them in clears them before it hands over.
      const int most = end_all - key0 - n * kUnit;
      if (most < kUnit && most % 16 != 0) {
        const int v = 2 * (n * kUnit / L::kTileKeys) + 1, first = most + n * kUnit % L::kTileKeys;  // ring number, row
        ok = __all_sync(0xffffffffu, ptx::wait_phase(&kv_full[v % L::kStages], (v / L::kStages) & 1, abort_flag, a.err,
                                                     kAttnWaitLoad));
        const unsigned at = sbase + L::kKv + v % L::kStages * L::kTile + first * 128;
        for (int i = r; i < (16 - most % 16) * 8 * L::kHalves; i += kRows)
          asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(at + i / 8 / L::kHalves * 128 +
                                                                      i / 8 % L::kHalves * L::kHalf + (i & 7) * 16),
                       "r"(0)
                       : "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      ptx::tc_wait_st();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&p_full[2 * w + (n & 1)]);
    }
    if (ok && mine > 0)
      ok = __all_sync(0xffffffffu, ptx::wait_phase(&pv_done[2 * w + ((mine - 1) & 1)], ((mine - 1) >> 1) & 1, abort_flag,
                                                   a.err, kAttnWaitMma));
    if (ok) {
      ptx::tc_fence_after();
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const long long t = q0 + tok;
      const int h = kvh * a.group + g;
      const long long row = t * a.heads + h;
      const bool parts = a.part_o != nullptr;
      // The rows leave through this warp's share of Q's place, 16 bytes a lane and
      // whole rows at a time (a lane that stores its own row alone touches 32
      // lines an instruction: 2000 cycles for a tile, now under 900).
      constexpr int kRowBytes = L::kQ / kRows, kChunks = kRowBytes / 16;
      const unsigned stage = sbase + w * L::kQ + (warp & 3) * 32 * kRowBytes;
      const unsigned long long to =
          parts ? reinterpret_cast<unsigned long long>(a.part_o + (split * a.total_q * a.heads + row) * a.head_size)
                : reinterpret_cast<unsigned long long>(static_cast<T*>(a.out) + t * a.out_token + h * a.out_head);
      const unsigned lives = __ballot_sync(0xffffffffu, live);
      auto put = [&](int chunk, unsigned x, unsigned y, unsigned z, unsigned u) {
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * kRowBytes + ((chunk ^ (lane & 7)) << 4)),
                     "r"(x), "r"(y), "r"(z), "r"(u)
                     : "memory");
      };
      // Rows of the stage to their places, 16 bytes a lane, eight loads before the stores.
      auto drain = [&](int from, int size) {
        __syncwarp();
        const int chunk = lane % kChunks, channel = from + chunk * (16 / size);
        constexpr int kEach = 32 / kChunks, kBatch = 8;
#pragma unroll
        for (int i = 0; i < kChunks; i += kBatch) {
          uint4 v[kBatch];
          unsigned long long dst[kBatch];
#pragma unroll
          for (int b = 0; b < kBatch; ++b) {
            const int r2 = (i + b) * kEach + lane / kChunks;
            dst[b] = __shfl_sync(0xffffffffu, to, r2);
            v[b] = lds16(stage + r2 * kRowBytes + ((chunk ^ (r2 & 7)) << 4));
          }
#pragma unroll
          for (int b = 0; b < kBatch; ++b) {
            const int r2 = (i + b) * kEach + lane / kChunks;
            if (((lives >> r2) & 1u) && channel < a.head_size)
              *reinterpret_cast<uint4*>(dst[b] + (unsigned long long)channel * size) = v[b];
          }
        }
        __syncwarp();
      };
      const bool blank = __any_sync(0xffffffffu, l == 0.0f);  // rows whose O means nothing
      auto take = [&](int from, auto count, float* v) {  // columns of O, divided by the row's sum
        constexpr int N = decltype(count)::value;
        if (mine > 0) {
#pragma unroll
          for (int e = 0; e < N; e += 32) ptx::tmem_ld32(o_addr + from + e, reinterpret_cast<unsigned*>(v) + e);
          ptx::tc_wait_ld();
        }
        if (blank) {
#pragma unroll
          for (int e = 0; e < N; ++e) v[e] = l == 0.0f ? 0.0f : v[e];
        }
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] *= inv;
      };
      // Keys that the products took in, masked ones among them: whole steps of 16, cleared behind the last that any row sees.
      const int last_key =
          min(end_all, key0 + (min(key1, work->end[w]) - key0 + 15) / 16 * 16);
      const float base = m == -INFINITY ? 0.0f : m * c;
      if (parts) {
#pragma unroll 1
        for (int from = 0; from < a.head_size; from += D / 2) {
          float v[D / 2];
          take(from, std::integral_constant<int, D / 2>{}, v);
          unsigned bad = 0;
          if (a.causal) {
            uint64_t zero = 0;  // stays 0 while all are finite
#pragma unroll
            for (int e = 0; e < D / 2; e += 2)
              if (from + e < a.head_size) zero = ptx::fma2(ptx::pair(v[e], v[e + 1]), 0, zero);
            float z0, z1;
            ptx::unpair(zero, z0, z1);
            bad = __ballot_sync(0xffffffffu, live && !(z0 == 0.0f && z1 == 0.0f));
          }
#pragma unroll
          for (int e = 0; e < D / 2; e += 4)
            put(e / 4, __float_as_uint(v[e]), __float_as_uint(v[e + 1]), __float_as_uint(v[e + 2]), __float_as_uint(v[e + 3]));
          if (bad) {
            __syncwarp();
            mend_rows<T>(a, bad, key0, last_key, sees, base, inv, t, h, k0, kvh, from, D / 2, stage, kRowBytes);
          }
          drain(from, 4);
        }
      } else {
        float v[D];
        take(0, std::integral_constant<int, D>{}, v);
        unsigned x[D / 2], bad = 0;
#pragma unroll
        for (int e = 0; e < D / 2; ++e) x[e] = ptx::pack16<BF16>(v[2 * e], v[2 * e + 1]);
        if (a.causal) {
          unsigned zero = 0;  // stays 0 while all are finite
#pragma unroll
          for (int e = 0; e < D / 2; ++e)
            if (2 * e < a.head_size) zero = ptx::times_zero<BF16>(x[e], zero);
          bad = __ballot_sync(0xffffffffu, live && (zero & 0x7fff7fffu) != 0);
        }
#pragma unroll
        for (int e = 0; e < D / 2; e += 4) put(e / 4, x[e], x[e + 1], x[e + 2], x[e + 3]);
        if (bad) {
          __syncwarp();
          mend_rows<T>(a, bad, key0, last_key, sees, base, inv, t, h, k0, kvh, 0, D, stage, kRowBytes);
        }
        drain(0, 2);
      }
      const float lse = (m == -INFINITY ? 0.0f : m * a.scale) + logf(l);
      if (live && a.part_o) a.part_lse[split * a.total_q * a.heads + row] = lse;
      if (live && !a.part_o && a.lse) a.lse[row] = lse;
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 4 * W) {
    ptx::tc_fence_after();
    ptx::tmem_free<L::kColumns>(*tmem_slot);
  }
}

// ------------------------------------------------------ one query a sequence ----

constexpr int kRowWarps = 4;       // warps that compute, each 16 keys of a stage: the MMA's M
constexpr int kRowThreads = 32 * (kRowWarps + 1);
constexpr int kStageKeys = 16 * kRowWarps;
constexpr int kRowHeads = 8;       // query heads of a CTA: the MMA's N

struct RowsArgs {
  const void* q = nullptr;
  long long q_seq = 0, q_head = 0;
  int prefix_len = 0;             // keys of the prefix that this kernel reads (0: attention_tc_kernel does)
  const int* suffix_lens = nullptr;
  int capacity = 0;
  int sequences = 0, heads = 0, kv_heads = 0, group = 0, head_size = 0;
  int blocks = 1;                 // blocks of kRowHeads heads of a group
  int splits = 1;
  float scale = 0.0f, scale_log2 = 0.0f;
  void* out = nullptr;            // the result (part_o == nullptr), or parts:
  long long out_seq = 0, out_head = 0;
  float* lse = nullptr;
  // merge: the splits of a row form a cluster, which joins them into the result;
  // else with part_o they leave parts.
  int merge = 0;
  float* part_o = nullptr;        // [splits x sequences x heads x head_size]
  float* part_lse = nullptr;      // [splits x sequences x heads]
  int wait = 0;                   // the launch before this one must be over when this one is
  int* err = nullptr;
};
struct RowsMaps {
  CUtensorMap pk, pv;  // prefix: (channel, KV head, key), 64 keys a copy
  CUtensorMap sk, sv;  // suffix: (channel, KV head, key, sequence), 16 keys a copy: none behind the length but in the last
};

// S stages.  D = 64: four, or two where more CTAs wait than SMs hold of those, five of
// which fit an SM instead of three (179 sessions of 18 keys, 16 KV heads: 21 us, then
// 16; two sessions of 7000 keys: 11.0 us, with two stages 12.1).  D = 128: two, three CTAs.
template <int D, int S>
struct RowsLayout {
  static constexpr int kHalf = kStageKeys * 128;  // 64 keys x 64 channels, 128-byte swizzle
  static constexpr int kTile = D / 64 * kHalf;
  static constexpr int kStages = S;
  static constexpr int kCtas = D == 64 && S == 2 ? 5 : 3;  // of an SM
  static constexpr int kBars = kStages * 2 * kTile;
  static constexpr int kMisc = kBars + 8 * 3 * kStages;
  static constexpr int kTotal = kMisc + 16 + 1024;
  static constexpr int kOut = kRowWarps * kRowHeads * (D + 4) * 4;  // the warps' sums, over the ring
  static constexpr int kFinal = kOut + 2 * kRowWarps * kRowHeads * 4;  // the CTA's sums, for its cluster
  static_assert(kFinal + (kRowHeads * D + 2 * kRowHeads) * 4 <= kBars, "joining the warps");
};

// D (m16n8) += A (m16k16) x B (k16n8), f32 accumulator.
template <bool BF16>
__device__ __forceinline__ void mma16816(float* d, unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                         unsigned b1) {
  if (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8 x 8 matrix of 16-bit values, lane (g, t) holding row g, columns 2t and 2t + 1: transposed.
__device__ __forceinline__ unsigned transpose8(unsigned x) {
  unsigned y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// One query token of one sequence, up to 8 of the heads that share a KV head.
// Warp 4 streams the keys through a ring of 64-key stages (TMA); warp w takes
// keys 16w .. 16w + 15 of a stage, and lane (g = lane / 4, t = lane % 4) reads
//   K rows g and g + 8, chunks 2t and 2t + 1 of each 64 channels (16 bytes each),
//   V rows 2t, 2t + 1, 2t + 8, 2t + 9, chunk g,
// all without bank conflicts under the 128-byte swizzle.  S^T = K Q^T sums over
// channels, whose order is free as long as Q has the same: the four words of a
// chunk serve as the k index of two MMAs.  O^T = V^T P^T needs pairs of keys in
// a word: two rows' words interleaved by prmt, so that the MMA of word r has
// channels 64h + 8g + 2r and + 2r + 1 as its rows g and g + 8.  P^T goes from
// S^T's layout to the operand's through movmatrix.  Bound: the bytes of K and V;
// the heads share them, so N = 8 serves groups up to 8 in one pass: one session's
// 65577 keys (8 KV heads of 128) take 44.5 us with the join, 6.0 TB/s of the 6.5 that a copy reaches, and the
// own keys of 256 sessions alone 83 us, 6.1 TB/s.  (Loads from global memory into
// registers needed the L1 for what was in flight: they ran at half the rate on an
// SM whose memory the tensor-core kernel had claimed.)
template <int D, int S, bool BF16>
__global__ void __launch_bounds__(kRowThreads, (RowsLayout<D, S>::kCtas))
    attention_rows_kernel(const RowsArgs a, const __grid_constant__ RowsMaps maps) {
  using L = RowsLayout<D, S>;
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  constexpr int KB = D / 32, VB = D / 64, NO = D / 16;
  extern __shared__ uint8_t sm_raw[];
  uint8_t* sm = sm_raw + ((1024 - (ptx::saddr(sm_raw) & 1023)) & 1023);
  const unsigned sbase = ptx::saddr(sm);
  uint64_t* k_full = reinterpret_cast<uint64_t*>(sm + L::kBars);
  uint64_t* v_full = k_full + L::kStages;
  uint64_t* empty = v_full + L::kStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + L::kMisc);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  unsigned id = blockIdx.x;
  const int split = id % a.splits;  // a merging call: the CTA's rank in its cluster
  id /= a.splits;
  const int kvh = id % a.kv_heads;
  id /= a.kv_heads;
  const int block = id % a.blocks, seq = id / a.blocks;
  const int head0 = kvh * a.group + block * kRowHeads, n_heads = min(kRowHeads, a.group - block * kRowHeads);
  ptx::griddep_launch();
  if (threadIdx.x == 0) {
    for (int s = 0; s < L::kStages; ++s) {
      ptx::mbar_init(&k_full[s], 1);
      ptx::mbar_init(&v_full[s], 1);
      ptx::mbar_init(&empty[s], kRowWarps);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  const int own = a.suffix_lens ? clamp_to(a.suffix_lens[seq], a.capacity) : 0;
  // Stages of 64 keys: the prefix's, then the sequence's own.
  const int ps = (a.prefix_len + kStageKeys - 1) / kStageKeys, all = ps + (own + kStageKeys - 1) / kStageKeys;
  const int s0 = (int)((long long)all * split / a.splits), s1 = (int)((long long)all * (split + 1) / a.splits);
  __syncthreads();

  if (warp == kRowWarps) {
    // ---- copies ----
    if (lane == 0) {
      bool ok = true;
      int n = 0;
      for (int s = s0; s < s1 && ok; ++s, ++n) {
        const int st = n % L::kStages;
        if (n >= L::kStages)
          ok = ptx::wait_phase(&empty[st], (n / L::kStages - 1) & 1, abort_flag, a.err, kAttnWaitFree);
        if (!ok) break;
        const bool prefix = s < ps;
        const int key0 = (prefix ? s : s - ps) * kStageKeys;
        const int copies = prefix ? 1 : min(kRowWarps, (own - key0 + 15) / 16);
        const unsigned bytes = prefix ? L::kTile : copies * (L::kTile / kRowWarps);
        for (int v = 0; v < 2; ++v) {
          uint64_t* bar = v ? &v_full[st] : &k_full[st];
          const unsigned dst = sbase + (2 * st + v) * L::kTile;
          ptx::mbar_expect_tx(bar, bytes);
          for (int h = 0; h < VB; ++h) {
            if (prefix)
              ptx::tma_load_3d(dst + h * L::kHalf, v ? &maps.pv : &maps.pk, h * 64, kvh, key0, bar);
            else
              for (int c = 0; c < copies; ++c)
                ptx::tma_load_4d(dst + h * L::kHalf + c * 2048, v ? &maps.sv : &maps.sk, h * 64, kvh, key0 + 16 * c, seq,
                                 bar);
          }
        }
      }
      for (int i = max(0, n - L::kStages); i < n; ++i) {  // copies in flight land before the CTA exits
        ptx::wait_phase(&k_full[i % L::kStages], (i / L::kStages) & 1, abort_flag, a.err, kAttnWaitLoad, false);
        ptx::wait_phase(&v_full[i % L::kStages], (i / L::kStages) & 1, abort_flag, a.err, kAttnWaitLoad, false);
      }
      if (a.wait && blockIdx.x == gridDim.x - 1) ptx::griddep_wait();
    }
    return;
  }

  unsigned q[KB][4];  // the B operand of S^T: head g, chunk 2t + (b & 1) of channels 64 (b / 2) ..
#pragma unroll
  for (int b = 0; b < KB; ++b) {
    const int c0 = 64 * (b >> 1) + 8 * (2 * t + (b & 1));
    uint4 v = make_uint4(0, 0, 0, 0);
    if (g < n_heads && c0 < a.head_size)
      v = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + seq * a.q_seq + (head0 + g) * a.q_head + c0);
    q[b][0] = v.x;
    q[b][1] = v.y;
    q[b][2] = v.z;
    q[b][3] = v.w;
  }
  float o[NO][4];
#pragma unroll
  for (int i = 0; i < NO; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};  // heads 2t, 2t + 1
  const float c = a.scale_log2;
  bool ok = true;
  const unsigned k_row = sbase + (16 * warp + g) * 128, v_row = sbase + (16 * warp + 2 * t) * 128;

  for (int s = s0, n = 0; s < s1; ++s, ++n) {
    const int st = n % L::kStages;
    const unsigned ph = (n / L::kStages) & 1;
    // Keys of this warp's 16 that exist; the rest of the stage holds what was there before.
    const int left = (s < ps ? a.prefix_len - s * kStageKeys : own - (s - ps) * kStageKeys) - 16 * warp;
    ok = __all_sync(0xffffffffu, ptx::wait_phase(&k_full[st], ph, abort_flag, a.err, kAttnWaitLoad));
    if (!ok) break;
    float sc[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // key g: heads 2t, 2t + 1; key g + 8: the same heads
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      const unsigned at = k_row + 2 * st * L::kTile + (b >> 1) * L::kHalf + (((2 * t + (b & 1)) ^ g) << 4);
      const uint4 k0 = lds16(at), k1 = lds16(at + 8 * 128);
      mma16816<BF16>(sc, k0.x, k1.x, k0.y, k1.y, q[b][0], q[b][1]);
      mma16816<BF16>(sc, k0.z, k1.z, k0.w, k1.w, q[b][2], q[b][3]);
    }
    if (g >= left) sc[0] = sc[1] = -INFINITY;
    if (g + 8 >= left) sc[2] = sc[3] = -INFINITY;
    // The maximum moves only when a score is 2^kSlack above it.
    const float x0 = fmaxf(sc[0], sc[2]), x1 = fmaxf(sc[1], sc[3]);
    if (__any_sync(0xffffffffu, x0 * c > m[0] * c + kSlack || x1 * c > m[1] * c + kSlack)) {
      float x[2] = {x0, x1};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) x[i] = fmaxf(x[i], __shfl_xor_sync(0xffffffffu, x[i], d));
        const float top = fmaxf(m[i], x[i]);
        const float f = top == m[i] ? 1.0f : ptx::ex2((m[i] - top) * c);  // 0 while the sums are empty
        m[i] = top;
        l[i] *= f;
#pragma unroll
        for (int k = 0; k < NO; ++k) {
          o[k][i] *= f;
          o[k][2 + i] *= f;
        }
      }
    }
    const float base0 = m[0] == -INFINITY ? 0.0f : m[0] * c, base1 = m[1] == -INFINITY ? 0.0f : m[1] * c;
    const float p0 = ptx::ex2(fmaf(sc[0], c, -base0)), p1 = ptx::ex2(fmaf(sc[1], c, -base1));
    const float p2 = ptx::ex2(fmaf(sc[2], c, -base0)), p3 = ptx::ex2(fmaf(sc[3], c, -base1));
    l[0] += p0 + p2;
    l[1] += p1 + p3;
    const unsigned b0 = transpose8(ptx::pack16<BF16>(p0, p1)), b1 = transpose8(ptx::pack16<BF16>(p2, p3));
    ok = __all_sync(0xffffffffu, ptx::wait_phase(&v_full[st], ph, abort_flag, a.err, kAttnWaitLoad));
    if (!ok) break;
#pragma unroll
    for (int h = 0; h < VB; ++h) {
      uint4 vx[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = 2 * t + (i & 1) + 8 * (i >> 1);
        const unsigned at = v_row + (2 * st + 1) * L::kTile + h * L::kHalf + ((i & 1) + 8 * (i >> 1)) * 128 + ((g ^ (key & 7)) << 4);
        vx[i] = key < left ? lds16(at) : make_uint4(0, 0, 0, 0);
      }
      const unsigned* v0 = reinterpret_cast<const unsigned*>(&vx[0]);
      const unsigned* v1 = reinterpret_cast<const unsigned*>(&vx[1]);
      const unsigned* v2 = reinterpret_cast<const unsigned*>(&vx[2]);
      const unsigned* v3 = reinterpret_cast<const unsigned*>(&vx[3]);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        mma16816<BF16>(o[4 * h + r], __byte_perm(v0[r], v1[r], 0x5410), __byte_perm(v0[r], v1[r], 0x7632),
                       __byte_perm(v2[r], v3[r], 0x5410), __byte_perm(v2[r], v3[r], 0x7632), b0, b1);
    }
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(&empty[st]);
  }

  // ---- join the warps, over the ring ----
  float* sm_o = reinterpret_cast<float*>(sm);  // [warp][head][D + 4]
  float* sm_m = sm_o + kRowWarps * kRowHeads * (D + 4);
  float* sm_l = sm_m + kRowWarps * kRowHeads;
  asm volatile("bar.sync 1, %0;" ::"n"(32 * kRowWarps) : "memory");  // every stage is used up
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], d);
    if (g == 0) {
      sm_m[warp * kRowHeads + 2 * t + i] = m[i];
      sm_l[warp * kRowHeads + 2 * t + i] = l[i];
    }
#pragma unroll
    for (int h = 0; h < VB; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *reinterpret_cast<float2*>(sm_o + (warp * kRowHeads + 2 * t + i) * (D + 4) + 64 * h + 8 * g + 2 * r) =
            make_float2(o[4 * h + r][i], o[4 * h + r][2 + i]);
  }
  asm volatile("bar.sync 1, %0;" ::"n"(32 * kRowWarps) : "memory");
  float* fin_o = reinterpret_cast<float*>(sm + L::kFinal);  // [head][D]: sums relative to the head's maximum
  float* fin_top = fin_o + kRowHeads * D;                   // the maximum (log2), and the sum of exponentials
  float* fin_sum = fin_top + kRowHeads;
  const bool failed = *abort_flag != 0;
  for (int e = threadIdx.x; e < n_heads * (D / 4) && !failed; e += 32 * kRowWarps) {
    const int h = e / (D / 4), ch0 = (e % (D / 4)) * 4;
    float top = -INFINITY, sum = 0.0f, v[4] = {};
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) top = fmaxf(top, sm_m[w * kRowHeads + h]);
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) {
      const float f = ptx::ex2((sm_m[w * kRowHeads + h] - base) * c);
      sum = fmaf(f, sm_l[w * kRowHeads + h], sum);
      const float4 x = *reinterpret_cast<const float4*>(sm_o + (w * kRowHeads + h) * (D + 4) + ch0);
      v[0] = fmaf(f, x.x, v[0]);
      v[1] = fmaf(f, x.y, v[1]);
      v[2] = fmaf(f, x.z, v[2]);
      v[3] = fmaf(f, x.w, v[3]);
    }
    if (a.merge) {
      *reinterpret_cast<float4*>(fin_o + h * D + ch0) = make_float4(v[0], v[1], v[2], v[3]);
      if (ch0 == 0) {
        fin_top[h] = top * c;
        fin_sum[h] = sum;
      }
      continue;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = sum == 0.0f ? 0.0f : v[i] * inv;
    const long long row = ((long long)split * a.sequences + seq) * a.heads + head0 + h;
    if (ch0 < a.head_size) {
      if (a.part_o)
        *reinterpret_cast<float4*>(a.part_o + row * a.head_size + ch0) = make_float4(v[0], v[1], v[2], v[3]);
      else
        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + seq * a.out_seq + (head0 + h) * a.out_head + ch0) =
            make_uint2(ptx::pack16<BF16>(v[0], v[1]), ptx::pack16<BF16>(v[2], v[3]));
    }
    if (ch0 == 0) {
      const float lse = base * a.scale + logf(sum);
      if (a.part_lse) a.part_lse[row] = lse;
      else if (a.lse) a.lse[row] = lse;
    }
  }
  if (!a.merge) return;

  // ---- join the cluster's CTAs, a share of the row each ----
  ptx::cluster_arrive();
  ptx::cluster_wait();
  for (int e = threadIdx.x * a.splits + split; e < n_heads * (D / 4) && !failed; e += 32 * kRowWarps * a.splits) {
    const int h = e / (D / 4), ch0 = (e % (D / 4)) * 4;
    const long long row = (long long)seq * a.heads + head0 + h;
    float top = -INFINITY;
    for (int s = 0; s < a.splits; ++s) top = fmaxf(top, ptx::remote_f32(ptx::map_rank(ptx::saddr(fin_top + h), s)));
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f, v[4] = {};
    for (int s = 0; s < a.splits; ++s) {
      const float f = ptx::ex2(ptx::remote_f32(ptx::map_rank(ptx::saddr(fin_top + h), s)) - base);
      const float4 x = ptx::remote_f32x4(ptx::map_rank(ptx::saddr(fin_o + h * D + ch0), s));
      sum = fmaf(f, ptx::remote_f32(ptx::map_rank(ptx::saddr(fin_sum + h), s)), sum);
      v[0] = fmaf(f, x.x, v[0]);
      v[1] = fmaf(f, x.y, v[1]);
      v[2] = fmaf(f, x.z, v[2]);
      v[3] = fmaf(f, x.w, v[3]);
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = sum == 0.0f ? 0.0f : v[i] * inv;
    if (ch0 < a.head_size)
      *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + seq * a.out_seq + (head0 + h) * a.out_head + ch0) =
          make_uint2(ptx::pack16<BF16>(v[0], v[1]), ptx::pack16<BF16>(v[2], v[3]));
    if (ch0 == 0 && a.lse) a.lse[row] = base * 0.6931471805599453f + logf(sum);
  }
  ptx::cluster_arrive();
  ptx::cluster_wait();  // the others' sums stay until they were read
}

// Joins the parts of a row: lse = log sum_s e^lse_s, out = sum_s e^(lse_s - lse) o_s,
// in a fixed order.  W warps per row, each taking every W-th part: for a session's
// 65577 keys in 37 parts the whole call takes 49.3 us with one warp, 44.5 with four.
// Bound: a chain of dependent loads, few rows having many parts.
struct JoinArgs {
  const int* q_off = nullptr;  // rows of [q_off[0], q_off[sequences]) only (null: all)
  int sequences = 0;
  long long tokens = 0;
  int heads = 0, head_size = 0, parts = 0;
  const float* part_o = nullptr;
  const float* part_lse = nullptr;
  void* out = nullptr;
  long long out_token = 0, out_head = 0;
  float* lse = nullptr;
};

constexpr int kJoinWarps = 4;

template <typename T, int W>
__global__ void __launch_bounds__(32 * kJoinWarps, 8) join_kernel(const JoinArgs a) {
  __shared__ float4 sm_o[kJoinWarps][32];
  __shared__ float sm_sum[kJoinWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long rows = a.tokens * a.heads, row = (long long)blockIdx.x * (kJoinWarps / W) + warp / W;
  const int part = warp % W, c = lane * 4;
  ptx::griddep_wait();
  const long long t = row / a.heads;
  const int h = (int)(row - t * a.heads);
  const bool live = row < rows && (!a.q_off || (t >= a.q_off[0] && t < a.q_off[a.sequences]));
  float top = -INFINITY, sum = 0.0f, o[4] = {};
  if (live) {
    for (int s = lane; s < a.parts; s += 32) top = fmaxf(top, a.part_lse[s * rows + row]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float base = top == -INFINITY ? 0.0f : top;
    const long long step = W * rows;
    const float* lse = a.part_lse + part * rows + row;
    const float* from = a.part_o + (part * rows + row) * a.head_size + (c < a.head_size ? c : 0);
#pragma unroll 4
    for (int s = part; s < a.parts; s += W, lse += step, from += step * a.head_size) {
      const float4 v = *reinterpret_cast<const float4*>(from);
      const float f = expf(*lse - base);
      sum += f;
      o[0] = fmaf(f, v.x, o[0]);
      o[1] = fmaf(f, v.y, o[1]);
      o[2] = fmaf(f, v.z, o[2]);
      o[3] = fmaf(f, v.w, o[3]);
    }
  }
  const float base = top == -INFINITY ? 0.0f : top;
  if (W > 1) {
    sm_o[warp][lane] = make_float4(o[0], o[1], o[2], o[3]);
    if (lane == 0) sm_sum[warp] = sum;
    __syncthreads();
    if (part != 0) return;
#pragma unroll
    for (int w = 1; w < W; ++w) {
      const float4 v = sm_o[warp + w][lane];
      sum += sm_sum[warp + w];
      o[0] += v.x;
      o[1] += v.y;
      o[2] += v.z;
      o[3] += v.w;
    }
  }
  if (!live) return;
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
void encode_kv(CUtensorMap* m, int dtype, const void* base, int head_size, int kv_heads, int64_t keys,
               const int64_t* stride, int box_keys) {
  const cuuint64_t dims[3] = {(cuuint64_t)head_size, (cuuint64_t)kv_heads, (cuuint64_t)keys};
  const cuuint64_t strides[2] = {map_stride(kv_heads, stride[1]), map_stride(keys, stride[0])};
  const cuuint32_t box[3] = {64, 1, (cuuint32_t)box_keys};
  encode_tensor_map(m, map_type(dtype), 3, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// The sequences' own K or V: (channel, KV head, key, sequence), 64 channels x 16 keys a copy.
void encode_suffix(CUtensorMap* m, int dtype, const void* base, int head_size, int kv_heads, int64_t keys,
                   int64_t sequences, const int64_t* stride) {
  const cuuint64_t dims[4] = {(cuuint64_t)head_size, (cuuint64_t)kv_heads, (cuuint64_t)keys, (cuuint64_t)sequences};
  const cuuint64_t strides[3] = {map_stride(kv_heads, stride[2]), map_stride(keys, stride[1]),
                                 map_stride(sequences, stride[0])};
  const cuuint32_t box[4] = {64, 1, 16, 1};
  encode_tensor_map(m, map_type(dtype), 4, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Launches in clusters of `cluster` CTAs, with `after` behind a kernel of this file that signals its dependents early.
template <typename... P, typename... A>
void launch_after(void (*kernel)(P...), unsigned grid, unsigned block, int shared, bool after, int cluster,
                  cudaStream_t stream, A&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = shared;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  if (after) {
    attrs[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attrs[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attrs[cfg.numAttrs].val.clusterDim.x = cluster;
    attrs[cfg.numAttrs].val.clusterDim.y = attrs[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  cfg.attrs = attrs;
  FA_CUDA(cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...));
}

template <int D, int W, bool BF16>
void launch_tc_as(const TcArgs& t, const TcMaps& maps, cudaStream_t stream) {
  using L = TcLayout<D, W>;
  const unsigned grid = (unsigned)t.tiles * t.kv_heads * t.splits;
  attention_tc_kernel<D, W, BF16><<<grid, L::kThreads, L::kTotal, stream>>>(t, maps);
  FA_CUDA(cudaGetLastError());
}
template <int D, int W>
void launch_tc_of(const TcArgs& t, const TcMaps& maps, int dtype, cudaStream_t stream) {
  dtype == FA_DTYPE_BF16 ? launch_tc_as<D, W, true>(t, maps, stream) : launch_tc_as<D, W, false>(t, maps, stream);
}
// W: tiles of a CTA, for which t.tiles was counted.
void launch_tc(const TcArgs& t, const TcMaps& maps, int w, int dtype, cudaStream_t stream) {
  if (t.head_size <= 64)
    w == 2 ? launch_tc_of<64, 2>(t, maps, dtype, stream) : launch_tc_of<64, 1>(t, maps, dtype, stream);
  else
    w == 2 ? launch_tc_of<128, 2>(t, maps, dtype, stream) : launch_tc_of<128, 1>(t, maps, dtype, stream);
}

template <int D, int S>
void launch_rows(const RowsArgs& r, const RowsMaps& maps, unsigned grid, bool after, int cluster, int dtype,
                 cudaStream_t stream) {
  launch_after(dtype == FA_DTYPE_BF16 ? attention_rows_kernel<D, S, true> : attention_rows_kernel<D, S, false>, grid,
               kRowThreads, RowsLayout<D, S>::kTotal, after, cluster, stream, r, maps);
}

void launch_join(const JoinArgs& j, int dtype, cudaStream_t stream) {
  const int w = j.parts > 8 ? kJoinWarps : 1;
  const unsigned grid = (unsigned)((j.tokens * j.heads * w + kJoinWarps - 1) / kJoinWarps);
  const bool bf16 = dtype == FA_DTYPE_BF16;
  launch_after(w > 1 ? (bf16 ? join_kernel<__nv_bfloat16, kJoinWarps> : join_kernel<__half, kJoinWarps>)
                     : (bf16 ? join_kernel<__nv_bfloat16, 1> : join_kernel<__half, 1>),
               grid, 32 * kJoinWarps, 0, true, 1, stream, j);
}

// Query rows as (channel, head of the group, KV head, token).
void encode_q(CUtensorMap* m, int dtype, const void* base, int head_size, int group, int kv_heads, int64_t tokens,
              const int64_t* stride, int tile_tokens) {
  const cuuint64_t dims[4] = {(cuuint64_t)head_size, (cuuint64_t)group, (cuuint64_t)kv_heads, (cuuint64_t)tokens};
  const cuuint64_t strides[3] = {map_stride(group, stride[1]), map_stride(kv_heads, stride[1] * group),
                                 map_stride(tokens, stride[0])};
  const cuuint32_t box[4] = {64, (cuuint32_t)group, 1, (cuuint32_t)tile_tokens};
  encode_tensor_map(m, map_type(dtype), 4, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

constexpr int kSms = 148;  // of a B200; workspace sizes must not depend on a device being there
// The kernel adds keys and the rows of a CTA's tiles to a token's number in 32 bits.
constexpr int64_t kMostSum = (1ll << 31) - 1024;
static_assert(2 * kRows <= 1024 && 2 * kKeys <= 1024, "sums of a token and a tile");
constexpr int kMaxCluster = 8;   // splits of attention_rows_kernel that a cluster joins
// Key tiles of a sequence up to which a CTA takes one tile of rows (W = 1): nine
// sequences of 100 to 1500 frames take 69 us so and 81 with W = 2, two prompts of
// 8192 tokens 531 us so and 502 with W = 2.
constexpr double kShort = 8.0;
constexpr double kStepUs = 1.8;  // one key tile against two tiles of rows, measured on long prompts

// Bytes of `parts` partial results of `rows` rows.
int64_t part_bytes(int64_t parts, int64_t rows, int head_size) { return parts * rows * (head_size + 4) * 4; }

// Rows of all partial results of a packed call together, at most: what bounds a
// workspace for any batch up to given sizes.  Ranges that fill the SMs two or
// three times over need fewer (188288 in 3 million random calls).
constexpr int64_t kMostPartRows = 192 * 1024;
constexpr int kMostSplits = 64;

// CTAs per KV head of a packed call with w tiles each, an upper bound (place_searched).
int64_t packed_tiles(int64_t total_q, int sequences, int group, int w) {
  return total_q / (w * (kRows / group)) + sequences;
}

// How a packed call is cut: tiles per CTA and key ranges.
struct PackedPlan {
  int w = 2, splits = 1;
};
PackedPlan packed_plan(int64_t total_q, int64_t total_k, int sequences, int heads, int kv_heads, int head_size) {
  PackedPlan p;
  const double steps = (double)total_k / sequences / kKeys;  // key tiles of a sequence, on average
  p.w = steps <= kShort ? 1 : 2;
  const double ctas = (double)packed_tiles(total_q, sequences, heads / kv_heads, p.w) * kv_heads;
  // The longest sequence is taken for 2.5 times the average: its CTAs' steps, or
  // all steps spread over the SMs, at kStepUs each; cutting the keys costs a
  // second kernel and the parts' bytes, written and read.  Chunks on histories of
  // 3001 to 20000 keys take 299 us uncut and 91 as cut here (in 4; 115 in 3, 105 in
  // 8); two tokens on 1749 keys 13.0 us with ranges of two tiles
  // allowed and 20.3 with no fewer than four.
  auto cost = [&](int s) {
    const double longest = std::max(1.0, (sequences > 1 ? 2.5 : 1.0) * steps / s);
    const double each = (p.w == 2 ? kStepUs : 0.7 * kStepUs) * (head_size <= 64 ? 0.6 : 1.0), sms = p.w == 2 ? kSms : 2 * kSms;
    const double parts = s > 1 ? 4.0 + 2.0 * s * total_q * heads * (head_size + 1) * 4 / 4e6 : 0.0;
    return std::max(longest, ctas * steps / sms) * each + ctas * s / sms * 1.5 + parts;
  };
  double best = cost(1);
  for (int s = 2; s <= kMostSplits && s * 2 <= steps && (double)s * total_q * heads <= kMostPartRows;
       s += s < 8 ? 1 : s / 4) {
    const double c = cost(s);
    if (c < best) {
      best = c;
      p.splits = s;
    }
  }
  return p;
}

// CTAs of a packed call.
int64_t packed_ctas(const fa_attention_packed_args& a) {
  const PackedPlan p = packed_plan(a.total_q, a.total_k, a.sequences, a.heads, a.kv_heads, a.head_size);
  return packed_tiles(a.total_q, a.sequences, a.heads / a.kv_heads, p.w) * a.kv_heads * p.splits;
}

// Bytes that serve every packed call of up to total_q queries and total_k keys.
int64_t packed_bound(int64_t total_q, int64_t total_k, int heads, int head_size) {
  const int64_t splits = std::min<int64_t>(kMostSplits, total_k / (2 * kKeys));
  if (splits < 2) return 0;
  const double rows = std::min((double)kMostPartRows, (double)splits * total_q * heads);
  return part_bytes(1, (int64_t)rows, head_size);
}

// How a shared-prefix call is cut.
struct SharedPlan {
  bool tc = false;      // the prefix on the tensor cores, for all sequences at once
  int tc_splits = 0;    // its key ranges
  int row_splits = 1;   // key ranges of attention_rows_kernel
  // Who brings the parts together: nobody (there is one), attention_rows_kernel
  // with its splits in clusters, or a join_kernel.
  enum { kOne, kMerge, kJoin } join = kOne;
  int parts() const { return tc_splits + (join == kJoin ? row_splits : 0); }  // partial results in the workspace
};
// CTAs of the rows kernel per SM that key ranges are cut for where a join_kernel
// follows: without the prefix's kernel beside it, and with it.
constexpr int kRowJoin = 2, kRowJoinTc = 8;

// Read by every sequence's CTAs on its own the prefix costs these bytes (of L2,
// mostly); the tensor-core kernel and what it leaves to join cost 15 to 20 us
// (thresholds of 40, 80 and 160 MB, measured over 60 calls: 9.5, 9.3, 9.2 us on average).
bool prefix_on_tc(int64_t prefix_len, int sequences, int kv_heads, int head_size) {
  return (double)sequences * prefix_len * kv_heads * head_size * 4 > 1.6e8 && sequences >= 4;
}

SharedPlan shared_plan(int64_t prefix_len, int64_t capacity, int sequences, int heads, int kv_heads, int head_size) {
  SharedPlan p;
  const int group = heads / kv_heads;
  p.tc = prefix_on_tc(prefix_len, sequences, kv_heads, head_size);
  if (p.tc) {
    // The two kernels run side by side, the prefix's bound by its MMAs and the own
    // keys' by their bytes: more key ranges end the prefix sooner, leave fewer SMs
    // to the own keys meanwhile (a CTA of the prefix fills an SM) and more parts to
    // join.  Microseconds: 1.7 a key tile of two tiles of rows (one: 0.7 of it, head
    // sizes up to 64: 0.6), own keys for 0.6 of the capacity at 6.2 TB/s, less what
    // the free SMs read by then, and the parts.  Fitted to 24 calls, each measured with
    // seven cuts: on average 2 % behind the best of them (filling the SMs with the
    // prefix: 10 %; 237 sessions on 11045 keys take 72 us so and 64 as chosen here).
    const int64_t rows = (int64_t)sequences * group, ctas = (rows + 2 * kRows - 1) / (2 * kRows) * kv_heads;
    const int64_t tiles = (prefix_len + kKeys - 1) / kKeys;
    const double tile_us = 1.7 * (rows > kRows ? 1.0 : 0.7) * (head_size <= 64 ? 0.6 : 1.0);
    const double own_us = 2.0 + 0.6 * 4.0 * sequences * capacity * kv_heads * head_size / 6.2e6;
    const double part_us = 0.7 * 8.0 * sequences * heads * head_size / 6e6;
    double best = 1e30;
    for (int64_t n = 1; n == 1 || (n <= kSms / ctas && 2 * n <= tiles + 1); ++n) {
      const double prefix_us = 2.5 + (double)((tiles + n - 1) / n) * tile_us;
      const double meanwhile = prefix_us * std::min(1.0, 1.2 * std::max<int64_t>(0, kSms - n * ctas) / kSms);
      const double us = prefix_us + std::max(0.0, own_us - meanwhile) + n * part_us;
      if (us < best) {
        best = us;
        p.tc_splits = (int)n;
      }
    }
  }
  const int64_t ctas = (int64_t)sequences * kv_heads * ((group + kRowHeads - 1) / kRowHeads);
  const int64_t stages = ((p.tc ? 0 : prefix_len) + capacity + kStageKeys - 1) / kStageKeys;
  // Without the prefix's parts a cluster joins the splits (a call of 19 sessions
  // with up to 804 keys: 18.6 us uncut, 12.9 us in clusters); long rows with few
  // CTAs are cut finer than a cluster, and a join_kernel is one launch more.
  const int64_t wanted = std::max<int64_t>(1, std::min(3 * kSms / ctas, stages / 3));
  if (!p.tc && wanted <= 2 * kMaxCluster) {
    while (p.row_splits < kMaxCluster && 2 * p.row_splits <= wanted) p.row_splits *= 2;
    p.join = p.row_splits > 1 ? SharedPlan::kMerge : SharedPlan::kOne;
  } else {
    p.row_splits = (int)std::max<int64_t>(1, std::min<int64_t>((p.tc ? kRowJoinTc : kRowJoin) * kSms / ctas, stages / 4));
    p.join = SharedPlan::kJoin;
  }
  return p;
}

// Bytes that serve every shared-prefix call up to these sizes: the parts of
// shared_plan, each at the most that its conditions leave, which grow with the
// sizes.  `rows` is the batch's query rows; a CTA of the prefix has 2 kRows of
// them, one of the rows kernel kRowHeads.
int64_t shared_bound(int64_t prefix_len, int64_t capacity, int sequences, int heads, int kv_heads, int head_size) {
  prefix_len = std::min<int64_t>(prefix_len, 1 << 30);
  capacity = std::min<int64_t>(capacity, 1 << 30);
  const double rows = std::min((double)sequences * heads, 2147483647.0);  // larger calls, and prefixes, are declined
  const auto parts = [&](double splits, double most) { return std::min(splits * rows, most); };
  double need = 0.0;
  const int64_t stages = (prefix_len + capacity + kStageKeys - 1) / kStageKeys;
  if (stages / 3 > 2 * kMaxCluster) need = parts(stages / 4, kRowJoin * kSms * kRowHeads);
  if (prefix_on_tc(prefix_len, sequences, kv_heads, head_size)) {
    const int64_t tiles = (prefix_len + kKeys - 1) / kKeys, own = (capacity + kStageKeys - 1) / kStageKeys;
    need = std::max(need, std::max(rows, parts((tiles + 1) / 2, kSms * 2 * kRows)) +
                              std::max(rows, parts(own / 4, kRowJoinTc * kSms * kRowHeads)));
  }
  return part_bytes(1, (int64_t)need, head_size);
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
  if (a->total_q >= (1ll << 31) || a->total_q * a->heads >= (1ll << 31) || a->total_k >= (1ll << 30) ||
      a->total_q + a->total_k > kMostSum)
    return kDeclined;
  if (a->total_q == 0 || a->sequences == 0) return kHandled;
  if (packed_ctas(*a) >= (1ll << 30)) return kDeclined;
  need(a->q && a->out && a->q_offsets && a->k_offsets, "null q, out, q_offsets or k_offsets");
  need(a->total_k == 0 || (a->k && a->v), "null k or v");
  need(aligned_to(4, {a->lse, a->q_offsets, a->k_offsets}), "lse or offsets not aligned to 4 bytes");
  const int64_t extents[2] = {a->total_q, a->heads};
  need(apart(a->out_stride, extents, a->head_size), "rows of out overlap");
  if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out)) return kDeclined;
  const auto rows = {a->total_q, (int64_t)a->heads}, keys = {a->total_k, (int64_t)a->kv_heads};
  if (!strides16(a->q_stride, rows) || !strides16(a->k_stride, keys) || !strides16(a->v_stride, keys) ||
      !strides16(a->out_stride, rows))
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
  if ((int64_t)a->sequences * a->heads >= (1ll << 31) || a->sequences > kMostSum || std::max(a->prefix_len, a->suffix_capacity) >= (1ll << 30) ||
      a->prefix_len + a->suffix_capacity >= (1ll << 30))
    return kDeclined;
  if (a->sequences == 0) return kHandled;
  need(a->q && a->out, "null q or out");
  need(a->prefix_len == 0 || (a->prefix_k && a->prefix_v), "null prefix_k or prefix_v");
  need(a->suffix_capacity == 0 || (a->suffix_k && a->suffix_v && a->suffix_lens),
       "null suffix_k, suffix_v or suffix_lens");
  need(aligned_to(4, {a->lse, a->suffix_lens}), "lse or suffix_lens not aligned to 4 bytes");
  const int64_t extents[2] = {a->sequences, a->heads};
  need(apart(a->out_stride, extents, a->head_size), "rows of out overlap");
  if (!aligned16(a->q) || !aligned16(a->prefix_k) || !aligned16(a->prefix_v) || !aligned16(a->suffix_k) ||
      !aligned16(a->suffix_v) || !aligned16(a->out))
    return kDeclined;
  const int64_t n = a->sequences, kv = a->kv_heads;
  const auto rows = {n, (int64_t)a->heads}, prefix = {a->prefix_len, kv}, suffix = {n, a->suffix_capacity, kv};
  if (!strides16(a->q_stride, rows) || !strides16(a->prefix_k_stride, prefix) || !strides16(a->prefix_v_stride, prefix) ||
      !strides16(a->suffix_k_stride, suffix) || !strides16(a->suffix_v_stride, suffix) || !strides16(a->out_stride, rows))
    return kDeclined;
  need(a->workspace_bytes >= attention_shared_workspace(a->prefix_len, a->suffix_capacity, a->sequences, a->heads,
                                                        a->kv_heads, a->head_size) &&
           (a->workspace_bytes == 0 || (a->workspace && aligned16(a->workspace))),
       "workspace smaller than fa_dev_attention_shared_workspace, or not on 16 bytes");
  return kHandled;
}

int64_t attention_packed_workspace(int64_t total_q, int64_t total_k, int sequences, int heads, int kv_heads,
                                   int head_size) {
  if (total_q <= 0 || sequences <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || heads / kv_heads > 64) return 0;
  const int splits = packed_plan(total_q, total_k, sequences, heads, kv_heads, head_size).splits;
  return splits > 1 ? part_bytes(splits, total_q * heads, head_size) : 0;
}
int64_t attention_shared_workspace(int64_t prefix_len, int64_t suffix_capacity, int sequences, int heads, int kv_heads,
                                   int head_size) {
  if (sequences <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || heads / kv_heads > 64) return 0;
  const SharedPlan p = shared_plan(prefix_len, suffix_capacity, sequences, heads, kv_heads, head_size);
  return part_bytes(p.parts(), (int64_t)sequences * heads, head_size);
}

int64_t attention_packed_workspace_bound(int64_t total_q, int64_t total_k, int heads, int kv_heads, int head_size) {
  if (total_q <= 0 || total_k <= 0 || heads <= 0 || kv_heads <= 0 || head_size <= 0 || heads % kv_heads) return 0;
  return packed_bound(total_q, total_k, heads, head_size);
}
int64_t attention_shared_workspace_bound(int64_t prefix_len, int64_t suffix_capacity, int sequences, int heads,
                                         int kv_heads, int head_size) {
  if (prefix_len < 0 || suffix_capacity < 0 || sequences <= 0 || heads <= 0 || kv_heads <= 0 || head_size <= 0 ||
      heads % kv_heads)
    return 0;
  return shared_bound(prefix_len, suffix_capacity, sequences, heads, kv_heads, head_size);
}

void prepare_dev_attention() {
  auto set = [](auto kernel, int bytes) {
    FA_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  };
  set(attention_rows_kernel<64, 4, false>, RowsLayout<64, 4>::kTotal);
  set(attention_rows_kernel<64, 4, true>, RowsLayout<64, 4>::kTotal);
  set(attention_rows_kernel<64, 2, false>, RowsLayout<64, 2>::kTotal);
  set(attention_rows_kernel<64, 2, true>, RowsLayout<64, 2>::kTotal);
  set(attention_rows_kernel<128, 2, false>, RowsLayout<128, 2>::kTotal);
  set(attention_rows_kernel<128, 2, true>, RowsLayout<128, 2>::kTotal);
  set(attention_tc_kernel<64, 1, false>, TcLayout<64, 1>::kTotal);
  set(attention_tc_kernel<64, 1, true>, TcLayout<64, 1>::kTotal);
  set(attention_tc_kernel<64, 2, false>, TcLayout<64, 2>::kTotal);
  set(attention_tc_kernel<64, 2, true>, TcLayout<64, 2>::kTotal);
  set(attention_tc_kernel<128, 1, false>, TcLayout<128, 1>::kTotal);
  set(attention_tc_kernel<128, 1, true>, TcLayout<128, 1>::kTotal);
  set(attention_tc_kernel<128, 2, false>, TcLayout<128, 2>::kTotal);
  set(attention_tc_kernel<128, 2, true>, TcLayout<128, 2>::kTotal);
}

void launch_attention_packed(const fa_attention_packed_args& a, int* err, cudaStream_t stream) {
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
  const PackedPlan plan = packed_plan(a.total_q, a.total_k, a.sequences, a.heads, a.kv_heads, a.head_size);
  t.tiles = (int)packed_tiles(a.total_q, a.sequences, t.group, plan.w);
  t.splits = plan.splits;
  t.causal = a.causal;
  t.scale = a.scale;
  t.scale_log2 = (float)(a.scale * 1.4426950408889634);
  t.out = a.out;
  t.out_token = a.out_stride[0];
  t.out_head = a.out_stride[1];
  t.lse = a.lse;
  t.err = err;
  t.q = a.q;
  t.k = a.k;
  t.v = a.v;
  t.q_token = a.q_stride[0];
  t.q_head = a.q_stride[1];
  t.k_token = a.k_stride[0];
  t.k_head = a.k_stride[1];
  t.v_token = a.v_stride[0];
  t.v_head = a.v_stride[1];
  if (t.splits > 1) {
    t.part_o = static_cast<float*>(a.workspace);
    t.part_lse = t.part_o + t.splits * a.total_q * a.heads * a.head_size;
  }
  TcMaps maps;
  encode_q(&maps.q, a.dtype, a.q, a.head_size, t.group, a.kv_heads, a.total_q, a.q_stride, t.tokens);
  if (a.total_k > 0) {
    const int keys = plan.w == 2 ? TcLayout<128, 2>::kTileKeys : TcLayout<128, 1>::kTileKeys;
    encode_kv(&maps.k, a.dtype, a.k, a.head_size, a.kv_heads, a.total_k, a.k_stride, keys);
    encode_kv(&maps.v, a.dtype, a.v, a.head_size, a.kv_heads, a.total_k, a.v_stride, keys);
  } else {
    maps.k = maps.v = maps.q;  // never used: no sequence has a key
  }
  launch_tc(t, maps, plan.w, a.dtype, stream);
  if (t.splits > 1) {
    JoinArgs j;
    j.q_off = a.q_offsets;
    j.sequences = a.sequences;
    j.tokens = a.total_q;
    j.heads = a.heads;
    j.head_size = a.head_size;
    j.parts = t.splits;
    j.part_o = t.part_o;
    j.part_lse = t.part_lse;
    j.out = a.out;
    j.out_token = a.out_stride[0];
    j.out_head = a.out_stride[1];
    j.lse = a.lse;
    launch_join(j, a.dtype, stream);
  }
}

void launch_attention_shared(const fa_attention_shared_args& a, int* err, cudaStream_t stream) {
  if (a.sequences == 0) return;
  const SharedPlan plan = shared_plan(a.prefix_len, a.suffix_capacity, a.sequences, a.heads, a.kv_heads, a.head_size);
  const int64_t rows = (int64_t)a.sequences * a.heads;
  const int group = a.heads / a.kv_heads, parts = plan.parts();
  float* part_o = parts ? static_cast<float*>(a.workspace) : nullptr;
  float* part_lse = parts ? part_o + parts * rows * a.head_size : nullptr;
  const float scale_log2 = (float)(a.scale * 1.4426950408889634);
  if (plan.tc) {
    TcArgs t;
    t.total_q = a.sequences;
    t.total_k = a.prefix_len;
    t.heads = a.heads;
    t.kv_heads = a.kv_heads;
    t.group = group;
    t.head_size = a.head_size;
    t.tokens = kRows / group;
    t.tiles = (a.sequences + 2 * t.tokens - 1) / (2 * t.tokens);
    t.splits = plan.tc_splits;
    t.scale = a.scale;
    t.scale_log2 = scale_log2;
    t.part_o = part_o;
    t.part_lse = part_lse;
    t.err = err;
    TcMaps maps;
    encode_q(&maps.q, a.dtype, a.q, a.head_size, group, a.kv_heads, a.sequences, a.q_stride, t.tokens);
    encode_kv(&maps.k, a.dtype, a.prefix_k, a.head_size, a.kv_heads, a.prefix_len, a.prefix_k_stride, kKeys);
    encode_kv(&maps.v, a.dtype, a.prefix_v, a.head_size, a.kv_heads, a.prefix_len, a.prefix_v_stride, kKeys);
    launch_tc(t, maps, 2, a.dtype, stream);
  }
  RowsArgs r;
  r.q = a.q;
  r.q_seq = a.q_stride[0];
  r.q_head = a.q_stride[1];
  r.prefix_len = plan.tc ? 0 : (int)a.prefix_len;
  r.suffix_lens = a.suffix_capacity > 0 ? a.suffix_lens : nullptr;
  r.capacity = (int)a.suffix_capacity;
  r.sequences = a.sequences;
  r.heads = a.heads;
  r.kv_heads = a.kv_heads;
  r.group = group;
  r.head_size = a.head_size;
  r.blocks = (group + kRowHeads - 1) / kRowHeads;
  r.splits = plan.row_splits;
  r.scale = a.scale;
  r.scale_log2 = scale_log2;
  r.out = a.out;
  r.out_seq = a.out_stride[0];
  r.out_head = a.out_stride[1];
  r.lse = a.lse;
  r.merge = plan.join == SharedPlan::kMerge;
  r.wait = plan.tc;
  if (plan.join == SharedPlan::kJoin) {
    r.part_o = part_o + plan.tc_splits * rows * a.head_size;
    r.part_lse = part_lse + plan.tc_splits * rows;
  }
  r.err = err;
  RowsMaps maps;
  if (r.prefix_len > 0) {
    encode_kv(&maps.pk, a.dtype, a.prefix_k, a.head_size, a.kv_heads, a.prefix_len, a.prefix_k_stride, kStageKeys);
    encode_kv(&maps.pv, a.dtype, a.prefix_v, a.head_size, a.kv_heads, a.prefix_len, a.prefix_v_stride, kStageKeys);
  }
  if (r.suffix_lens) {
    encode_suffix(&maps.sk, a.dtype, a.suffix_k, a.head_size, a.kv_heads, a.suffix_capacity, a.sequences, a.suffix_k_stride);
    encode_suffix(&maps.sv, a.dtype, a.suffix_v, a.head_size, a.kv_heads, a.suffix_capacity, a.sequences, a.suffix_v_stride);
  }
  const unsigned grid = (unsigned)((int64_t)a.sequences * a.kv_heads * r.blocks * r.splits);
  const int cluster = r.merge ? plan.row_splits : 1;
  if (a.head_size > 64)
    launch_rows<128, 2>(r, maps, grid, plan.tc, cluster, a.dtype, stream);
  else if (grid > (unsigned)(RowsLayout<64, 4>::kCtas * kSms))
    launch_rows<64, 2>(r, maps, grid, plan.tc, cluster, a.dtype, stream);
  else
    launch_rows<64, 4>(r, maps, grid, plan.tc, cluster, a.dtype, stream);
  if (plan.join == SharedPlan::kJoin) {
    JoinArgs j;
    j.tokens = a.sequences;
    j.heads = a.heads;
    j.head_size = a.head_size;
    j.parts = parts;
    j.part_o = part_o;
    j.part_lse = part_lse;
    j.out = a.out;
    j.out_token = a.out_stride[0];
    j.out_head = a.out_stride[1];
    j.lse = a.lse;
    launch_join(j, a.dtype, stream);
  }
}

ErrorWord take_error_word(int device, cudaStream_t stream) {
  std::lock_guard<std::mutex> lk(g_words_mu);
  std::vector<int>& users = g_word_users[device];
  users.resize(kErrorWords);
  ErrorWord w;
  w.device = device;
  w.slot = (int)(std::min_element(users.begin(), users.end()) - users.begin());
  void* p = nullptr;
  FA_CUDA(cudaGetSymbolAddress(&p, g_dev_errors));
  w.word = static_cast<int*>(p) + w.slot;
  if (users[w.slot] == 0) {
    FA_CUDA(cudaMemsetAsync(w.word, 0, sizeof(int), stream));
    FA_CUDA(cudaStreamSynchronize(stream));
  }
  ++users[w.slot];
  return w;
}

void give_error_word(const ErrorWord& w) {
  if (w.word == nullptr) return;
  std::lock_guard<std::mutex> lk(g_words_mu);
  --g_word_users[w.device][w.slot];
}

int read_error_word(const ErrorWord& w, cudaStream_t stream) {
  FA_CUDA(cudaDeviceSynchronize());
  int code = 0;
  FA_CUDA(cudaMemcpyAsync(&code, w.word, sizeof(code), cudaMemcpyDeviceToHost, stream));
  FA_CUDA(cudaStreamSynchronize(stream));
  if (code != 0) {
    FA_CUDA(cudaMemsetAsync(w.word, 0, sizeof(int), stream));
    FA_CUDA(cudaStreamSynchronize(stream));
  }
  return code;
}

namespace {
// A wait that nothing ends.
__global__ void fault_test_kernel(int* err) {
  __shared__ uint64_t bar;
  __shared__ int abort_flag;
  ptx::mbar_init(&bar, 1);
  abort_flag = 0;
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  ptx::wait_phase(&bar, 0, &abort_flag, err, kAttnWaitTest);
}
}  // namespace

void launch_fault_test(int* err, cudaStream_t stream) {
  fault_test_kernel<<<1, 1, 0, stream>>>(err);
  FA_CUDA(cudaGetLastError());
}

}  // namespace fa
