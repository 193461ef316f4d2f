// The device-pointer operators behind fa_dev_* (dev_attention.cu, dev_logits.cu).
// Argument structs are the C ABI's; the launchers expect them checked.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <initializer_list>

#include "../../include/funasr_cuda.h"
#include "fa_common.h"

namespace fa {

// The structs as hosts in other languages lay them out: no padding.
static_assert(sizeof(fa_attention_packed_args) == 184 && sizeof(fa_attention_shared_args) == 232 &&
                  sizeof(fa_logits_args) == 168,
              "argument struct layout");

// Whether all addresses are multiples of `size`, which the device faults without.
inline bool aligned_to(uintptr_t size, std::initializer_list<const void*> addresses) {
  for (const void* p : addresses)
    if (reinterpret_cast<uintptr_t>(p) % size != 0) return false;
  return true;
}

// kHandled, or kDeclined for sizes and alignments outside the kernels; throws
// on inconsistent arguments.  Host checks only: no device is needed.
int check_attention_packed(const fa_attention_packed_args* a);
int check_attention_shared(const fa_attention_shared_args* a);
int check_logits(const fa_logits_args* a);

int64_t attention_packed_workspace(int64_t total_q, int64_t total_k, int sequences, int heads, int kv_heads,
                                   int head_size);
int64_t attention_shared_workspace(int64_t prefix_len, int64_t suffix_capacity, int sequences, int heads, int kv_heads,
                                   int head_size);

int64_t attention_packed_workspace_bound(int64_t total_q, int64_t total_k, int heads, int kv_heads, int head_size);
int64_t attention_shared_workspace_bound(int64_t prefix_len, int64_t suffix_capacity, int sequences, int heads,
                                         int kv_heads, int head_size);

// `err`: the backend's error word.
void launch_attention_packed(const fa_attention_packed_args& a, int* err, cudaStream_t stream);
void launch_attention_shared(const fa_attention_shared_args& a, int* err, cudaStream_t stream);
void launch_adjust_logits(const fa_logits_args& a, int* err, cudaStream_t stream);

// Function attributes of these kernels on the current device; before any launch.
void prepare_dev_attention();
void prepare_dev_logits();

// A backend's error word, which a bounded wait of its kernels that gives up
// sets; `stream` is the backend's, the device the current one.
struct ErrorWord {
  int device = 0, slot = 0;
  int* word = nullptr;
};
ErrorWord take_error_word(int device, cudaStream_t stream);
void give_error_word(const ErrorWord& w);
// Waits for the device, then the word (0: no bounded wait gave up), cleared by the read.
int read_error_word(const ErrorWord& w, cudaStream_t stream);
// Enqueues a bounded wait that nothing ends.
void launch_fault_test(int* err, cudaStream_t stream);

}  // namespace fa
