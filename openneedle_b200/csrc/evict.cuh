// Eviction from a KV cache by accumulated attention weight: parameters and
// launch (evict.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace nb200 {

struct Evict {
    int batch, kvheads, capacity, out_capacity, keep, first, recent;
    int row_bytes;                        // bytes of one K or V row
    const char *k, *v;
    long long ks[3], vs[3];               // bytes: batch, KV head, key
    const float *kscale, *vscale;         // INT8 caches (null otherwise)
    long long kss[3], vss[3];             // elements
    const float *weights;
    long long ws[3];
    const int *lengths;
    char *ko, *vo;
    long long kos[3], vos[3];
    float *kscale_o, *vscale_o;
    long long ksos[3], vsos[3];
    float *weights_o;
    long long wos[3];
    int *indices;                         // [batch][kvheads][keep]
    int *lengths_o;
    bool in_place;                        // the outputs are the inputs
};

bool launch_evict(const Evict &e, cudaStream_t st);

}  // namespace nb200
