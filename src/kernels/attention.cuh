// Softmax attention over whole prompts that are packed one behind the other, with grouped heads, and its backward
// pass.  The reference has no model code.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace mgk {
namespace attn {

constexpr int kMaxDim = 128;

// [tokens, heads, dim] of 16-bit numbers: `row` and `head` are strides in elements, the innermost one is 1
struct Tensor {
    void* p;
    int64_t row, head;
};

struct Problem {
    bool fp16;           // else bf16
    int tokens;          // rows of every tensor
    int heads, kv_heads; // heads a multiple of kv_heads
    int dim;             // a multiple of 8, at most kMaxDim
    const int* cu;       // [seqs + 1] on the device: sequence s holds rows cu[s] .. cu[s + 1]; null: one of all rows
    int seqs;
    bool causal;
    float scale;         // > 0
    int* error_flag;     // set to 1 when a wait inside a kernel runs out; may be null
};

// out = softmax(scale q k^T) v, lse[head * tokens + row] = log of the sum of exponentials (natural)
cudaError_t launch_forward(const Problem& p, Tensor q, Tensor k, Tensor v, Tensor out, float* lse, cudaStream_t stream);

// `workspace`: backward_workspace(p) bytes, 16-byte aligned
size_t backward_workspace(const Problem& p);
cudaError_t launch_backward(const Problem& p, Tensor dout, Tensor q, Tensor k, Tensor v, Tensor out, const float* lse,
                            Tensor dq, Tensor dk, Tensor dv, void* workspace, cudaStream_t stream);

}  // namespace attn
}  // namespace mgk
