// decode_fp8_block.hip -- the decode kernels over fp8 pools with one scale a tile
// (v_mfma_f32_16x16x32_bf16).
#include "decode_stream.hpp"

namespace rkv {

Launch decode_fp8_block(int D, int G, int P, DecodeMode mode) {
  return pick_d<uint8_t, RKV_FP8_BLOCK>(D, G, P, mode);
}

}  // namespace rkv
