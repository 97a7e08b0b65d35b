// One AdamW step over a list of tensors.  The reference has no optimizer (it is a pure communication
// library).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace mgk {
namespace adamw {

constexpr int kBlock = 256;  // elements that share one scale where moments are kept in 8 bits

struct Tensor {
    void* p;        // parameters, float32 or bf16, updated in place
    const void* g;  // gradients, float32 or bf16
    void* copy;     // bf16 copy of the updated parameters, or null
    uint64_t n;
    uint64_t block;  // first block of kBlock elements in the moment buffers
};

struct Step {
    bool p_bf16, g_bf16;
    int bits;  // 32: m and v float32; 8: m and r = sqrt(v) as e4m3 with a float32 scale per block
    void *m, *v;
    float *m_scale, *v_scale;
    double lr, beta1, beta2, eps, weight_decay, grad_scale, step;
    // float32 numbers on the device that take the place of the ones above, or null
    const float *lr_dev, *grad_scale_dev, *step_dev;
};

cudaError_t launch(const Tensor* tensors, int count, const Step& s, cudaStream_t stream);

}  // namespace adamw
}  // namespace mgk
