// serve_kernels.cu -- the "serve" module image (sm_100a cubin): a batch of
// requests that share a prompt.  Page plan, rotary positions with the cache
// write, attention over the shared prefix and each request's own pages.
// None of them has a counterpart in the reference, which decodes one
// sequence at a time.
#include "serve_plan.cuh"
#include "serve_rotary.cuh"
#include "serve_attn.cuh"
#include "serve_attn_tc.cuh"
