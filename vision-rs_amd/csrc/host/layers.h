// What the entry points of the transformer-layer operators share: checks of
// arguments, and the launch.
#pragma once
#include "vrs_internal.h"

namespace vrs {

inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

inline int check_type(int dtype, const char* what) {
  if (dtype == VRS_BF16 || dtype == VRS_F32) return VRS_OK;
  return fail(VRS_EUNSUPPORTED, "%s: dtype %d (VRS_BF16 or VRS_F32)", what, dtype);
}

// Element types need their own alignment whatever the kernel.
inline int check_ptr(const void* p, size_t es, const char* what, const char* name) {
  if (!p) return fail(VRS_EINVAL, "%s: null %s", what, name);
  if (!aligned(p, es)) return fail(VRS_EBADSHAPE, "%s: %s is not aligned to its elements", what, name);
  return VRS_OK;
}

// Whether no two (row, head) of an output share an element: heads inside a row's stride, or rows
// inside a head's.
inline bool apart(int64_t ld, int64_t hd, int64_t rows, int64_t heads, int64_t dim) {
  if (rows <= 1 && heads <= 1) return true;
  if (rows <= 1) return hd >= dim;
  if (heads <= 1) return ld >= dim;
  return (hd >= dim && ld >= (heads - 1) * hd + dim) || (ld >= dim && hd >= (rows - 1) * ld + dim);
}

inline int check_seqs(const vrs_seqs* s, const char* what) {
  if (s->n < 0) return fail(VRS_EBADSHAPE, "%s: %d sequences", what, s->n);
  if (!s->q_start) return fail(VRS_EINVAL, "%s: null q_start", what);
  if (s->max_q < 0 || s->max_k < 0) return fail(VRS_EINVAL, "%s: negative max_q or max_k", what);
  return VRS_OK;
}

inline int launch(vrs_ctx* ctx, const char* name, dim3 grid, dim3 block, uint32_t lds, void* args, void* stream) {
  hipFunction_t f;
  if (int rc = get_fn(ctx, name, &f)) return rc;
  void* params[] = {args};
  hipError_t e = hipModuleLaunchKernel(f, grid.x, grid.y, grid.z, block.x, block.y, block.z, lds,
                                       static_cast<hipStream_t>(stream), params, nullptr);
  if (e != hipSuccess) return fail(VRS_EHIP, "launch %s: %s", name, hipGetErrorString(e));
  return VRS_OK;
}

// What vrs_attention refuses of a descriptor and sequences (layers.cpp).
int check_attention(const vrs_attention_desc* d, const vrs_seqs* seqs, const char* what);
// Its buffers: there, aligned, and out none of the inputs.
int check_attention_buffers(const vrs_attention_desc* d, const void* q, const void* k, const void* v, const void* out,
                            const char* what);

}  // namespace vrs
