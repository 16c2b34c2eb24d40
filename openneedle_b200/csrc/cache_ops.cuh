// The stateless attention call of the C ABI for other files of the library.
#pragma once
#include <cuda_runtime.h>

#include "../../include/needle2_b200.h"

namespace nb200 {

// Workspace bytes of a call, or -1 (with the error set); the call itself.
long long prefix_attention_workspace(const needle2_prefix_attention_args &a);
// At least the bytes of every call of one token a sequence, without weights, of up to
// a.batch sequences and a.capacity own keys, -1 (with the error set) for sizes refused.
long long prefix_attention_workspace_most(const needle2_prefix_attention_args &a);
bool prefix_attention(const needle2_prefix_attention_args &a, void *workspace, long long bytes, cudaStream_t st);

}  // namespace nb200
