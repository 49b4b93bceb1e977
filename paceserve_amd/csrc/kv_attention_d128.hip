// Attention with head_dim 128.
#include "attention.h"

namespace pace_kv {

const void* attention_kernel_d128(int type, int format, uint32_t tile_rows) {
  return pick_attention<128>(type, format, tile_rows);
}

}  // namespace pace_kv
