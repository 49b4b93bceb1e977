// Attention with head_dim 64.
#include "attention.h"

namespace pace_kv {

const void* attention_kernel_d64(int type, int format, uint32_t tile_rows) {
  return pick_attention<64>(type, format, tile_rows);
}

}  // namespace pace_kv
