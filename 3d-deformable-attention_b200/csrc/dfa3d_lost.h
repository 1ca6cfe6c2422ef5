// What an epilogue stores where a wait has run out (dfa3d_tcgen05.cuh: no sound run waits so long): a word that is NaN as one 32-bit
// number and as two of either 16-bit type, in all columns that it would have made of what did not come, so that no part of it can be
// taken for a result.  A warp that has given up hands nothing over any more: its count stays short, whoever waits for it gives up
// too, and no accumulator is summed into while another warp reads it.
#pragma once
#include <stdint.h>

namespace dfa3d {

constexpr uint32_t kLost = 0x7fffffffu;

}  // namespace dfa3d
