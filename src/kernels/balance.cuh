// Balance loss of a mixture-of-experts router with the pairs per expert and the gradient of the logits.
// The reference has no model code.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace mgk {
namespace balance {

constexpr int kMaxExperts = 1024;
constexpr int kMaxTop = 64;
constexpr int kMaxPartials = 48;

// float [E] sums of probabilities, then int32 [E] pairs per expert, then int32 tokens that count, padded to 4
__host__ __device__ constexpr int partial_words(int experts) { return (2 * experts + 1 + 3) / 4 * 4; }

struct Router {
    const void* logits;  // [tokens, experts], rows `ld` elements apart
    bool bf16;
    int64_t ld;
    const void* idx;     // [tokens, top] experts of each token, contiguous
    bool idx64;
    const uint8_t* mask; // [tokens]: 0 = the token does not count; null = all count
    int tokens, experts, top;
};

// The workspace holds kMaxPartials such records and two float32 a token (a row's maximum and reciprocal sum).
size_t workspace_bytes(int tokens, int experts);
// Number of partial sums that launch_stats writes for this size (1 .. kMaxPartials).
int partials(int tokens, int experts);
cudaError_t launch_stats(const Router& r, void* workspace, cudaStream_t stream);

struct Result {
    float coef;
    float* loss;    // [1]
    int* counts;    // [experts]
    void* dlogits;  // [tokens, experts], the type of the logits or float32, rows `ldd` elements apart; or null
    bool d_bf16;
    int64_t ldd;
    bool accumulate;
};
// `n_partials` partial sums as launch_stats wrote them (one, if they were added up over ranks meanwhile) and the
// workspace that it wrote for the same router.  `follows_stats`: launch_stats is the stream's last launch.
cudaError_t launch_grad(const Router& r, const void* partial, int n_partials, const void* workspace, const Result& out,
                        bool follows_stats, cudaStream_t stream);
// Both in a single launch for a problem that one cluster handles.
bool is_small(int tokens, int experts);
cudaError_t launch_small(const Router& r, void* workspace, const Result& out, cudaStream_t stream);

}  // namespace balance
}  // namespace mgk
