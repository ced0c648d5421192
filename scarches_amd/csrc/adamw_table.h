// Entries of the table that sca_adamw_step walks; layout of include/scarches_hip.h.
#pragma once
#include <stdint.h>

extern "C" {
typedef struct {
    void* p; const void* g; void* m; void* v;
    float* m_scale; float* v_scale;
    long long n;
    int64_t* step;
    float weight_decay;
    int32_t dtype, vec, id;
} sca_adamw_tensor;
typedef struct {
    int32_t tensor, index;
} sca_adamw_chunk;
}
