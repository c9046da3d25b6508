// Host interface of the split decode (split_decode.cuh), compiled apart from
// the ABI unit so that its instantiations build in parallel.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/cpu_attention_b200.h"

namespace ca {

struct SplitCall {
  const void* q;
  long long q_stride;
  const void* kc;
  const void* vc;
  const float* ks;
  const float* vs;
  long long num_blocks;
  const int32_t* lens;
  long long n_new;  // tokens already appended at lens[i]
  const int32_t* page_table;
  long long table_width;
  void* out;
  float* lse;
  long long batch, heads, kv_heads;
  int head_dim;
  long long page;
  int q_dtype, cache_dtype;
  long long left, sinks;
  float c;
  void* workspace;
  int32_t* status;
};

size_t split_workspace_bytes(int head_dim, int sms);
cudaError_t split_launch(const SplitCall& c, int sms, int device, cudaStream_t stream);

// ca_abi.cu: records the error and returns CA_ECUDA; the current device's SMs
int host_cuda_fail(cudaError_t e, const char* what);
int host_sms(int* sms);

}  // namespace ca
