// Argument check shared by the entry points that take a kvm_kv_layout.
#pragma once

#include "runtime.h"

namespace kvm {

inline int check_kv_layout(const kvm_kv_layout* L) {
  if (!L) return fail(KVM_ERR_INVALID_ARG, "kv layout is NULL");
  if (L->block_size < 1 || L->width <= 0 || L->width % 8 || L->num_pages <= 0 ||
      L->layer < 0 || L->token_stride < L->width || L->token_stride % 8 ||
      L->page_stride % 8 || L->layer_stride % 8 || L->kv_stride % 8)
    return fail(KVM_ERR_INVALID_ARG,
                "kv layout: need block_size >= 1, width % 8 == 0, 16-byte aligned "
                "strides and token_stride >= width");
  return KVM_OK;
}

}  // namespace kvm
