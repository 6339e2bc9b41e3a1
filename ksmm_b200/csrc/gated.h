// Host interface of the gated layer's kernels: the product of the two halves (gated.cu) and the factor that
// forms it in its epilogue (tc_gated.cu).
#pragma once

#include "common.cuh"

namespace ksmm {

constexpr int kGatedWaits = 90;  // codes of tc_gated.cu's bounded waits: 90 to 95

// h = act(g) * u.  g and u: `lines` lines of `len` elements with stride `ld`, u after g; h has stride `h_ld`.
int launch_gate(const void* gu, int64_t ld, void* h, int64_t h_ld, int64_t lines, int64_t len, int dtype, int act,
                cudaStream_t stream);
// the same in the other layout: h is (len, lines) without gaps
int launch_gate_turn(const void* gu, int64_t ld, void* h, int64_t lines, int64_t len, int dtype, int act, cudaStream_t stream);
// dg = dh u act'(g), du = dh act(g); `out` holds dg and, out_half elements after it, du (stride ld).
// bias_grad != NULL: also the sums of every line of dg, then of du, (2, lines) in the tensors' type
int launch_gate_backward(const void* gu, int64_t ld, const void* dh, int64_t dh_ld, void* out, int64_t out_half, int64_t lines,
                         int64_t len, int dtype, int act, void* bias_grad, cudaStream_t stream);

// Can the 16-bit tensor-core kernel run the last factor (pattern q) and the product in one launch?  Pointers and
// row strides of what it reads and writes are multiples of 16 bytes, except a batch-last output's.
bool tc_gated_fits(const int32_t* q, int64_t batch, int dtype, int in_last, int out_last);
// p: the factor with stacked weights, bias and (group_shared_input == 0) input; p.out = h, p.activation = the
// gate's.  halves != NULL: both halves are stored there too (batch-last rows halves_ld apart).  turn: the problem's
// output is batch-last, but h is stored batch-first, element by element (for small batches, in place of a transpose).
int tc_gated_launch(const Problem& p, void* halves, int64_t halves_ld, bool turn, cudaStream_t stream);
// p.out = the sum of both halves of a factor with a stacked batch-last input and stacked weights, no bias; for what
// tc_gated_fits says
int tc_gated_sum(const Problem& p, cudaStream_t stream);

}  // namespace ksmm
