// What the kernels of the 8-bit block cache share: the view of the pool and its host checks.
#pragma once

#include "ctmi_device.h"
#include "ctmi_host.h"

namespace ctmi {

inline int check_kv_blocks(const ctmi_kv_blocks* b) {
  CTMI_REQUIRE(b != nullptr, CTMI_ERR_VALUE, "blocks is NULL");
  CTMI_REQUIRE(b->num_blocks >= 0 && b->num_blocks < (1ll << 31) && b->kv_heads >= 1, CTMI_ERR_VALUE,
               "bad pool: %lld blocks, %d heads", (long long)b->num_blocks, b->kv_heads);
  CTMI_REQUIRE(b->code_dtype == CTMI_F8E4M3 || b->code_dtype == CTMI_I8, CTMI_ERR_UNSUPPORTED,
               "codes must be float8_e4m3fn or int8");
  CTMI_REQUIRE(b->head_dim == 64 || b->head_dim == 128 || b->head_dim == 256, CTMI_ERR_UNSUPPORTED,
               "head_dim must be 64, 128 or 256, got %d", b->head_dim);
  CTMI_REQUIRE(b->block_size >= 16 && b->block_size <= 256 && b->block_size % 16 == 0, CTMI_ERR_UNSUPPORTED,
               "block_size must be a multiple of 16 up to 256, got %d", b->block_size);
  CTMI_REQUIRE(b->num_blocks == 0 || (b->key && b->value && b->key_scale && b->value_scale), CTMI_ERR_VALUE,
               "NULL tensor in blocks");
  CTMI_REQUIRE(((uintptr_t)b->key | (uintptr_t)b->value) % 16 == 0, CTMI_ERR_VALUE,
               "key and value codes must be 16-byte aligned");
  return CTMI_OK;
}

}  // namespace ctmi
