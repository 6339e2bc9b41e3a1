// Host interface of the gated layer's kernels: the product of the two halves (gated.cu) and the factor that
// forms it in its epilogue (tc_gated.cu).
#pragma once

#include "common.cuh"

namespace ksmm {

// h = act(g) * u.  g and u: `lines` lines of `len` elements with stride `ld`, u after g; h has stride `h_ld`.
int launch_gate(const void* gu, int64_t ld, void* h, int64_t h_ld, int64_t lines, int64_t len, int dtype, int act,
                cudaStream_t stream);
// dg = dh u act'(g), du = dh act(g); `out` holds dg and, out_half elements after it, du (stride ld)
int launch_gate_backward(const void* gu, int64_t ld, const void* dh, int64_t dh_ld, void* out, int64_t out_half, int64_t lines,
                         int64_t len, int dtype, int act, cudaStream_t stream);

}  // namespace ksmm
