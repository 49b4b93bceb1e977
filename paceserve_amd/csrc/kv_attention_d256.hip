// Attention with head_dim 256.
#include "attention.h"

namespace pace_kv {

const void* attention_kernel_d256(int type, int format, uint32_t tile_rows) {
  return pick_attention<256>(type, format, tile_rows);
}

}  // namespace pace_kv
