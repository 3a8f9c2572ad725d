// gemm_tile.h instantiated for codes of 8 bits (two k-contiguous operands): Y = X W^T with a scale per row of each, and its
// gate/up form.  Bound by the matrix cores at many rows (8192 x 24576 x 4096 with SwiGLU: 651 - 693 us, 2.4 - 2.5 POP/s, where a
// plain library product of 16384 cubed reaches 2.4), by the weights' stream and a k-tile's latency at few (32 x 4096 x 12288:
// 11.3 - 12.0 us and 3 - 4 for the join, 4.4 TB/s).
#include "gemm_tile.h"

namespace q3gemm {

// The waves of a tile: eight wherever its loads can be dealt out to eight.  A k-tile's matrix work is half of the 16-bit
// kernels' per code, so what a wave waits for shows: 128 x 128 on four waves took 28.6 us for 1024 x 4096 x 4096, on eight 23.4
// (64 x 64, 256 x 4096 x 4096: 12.7 and 11.2), a third stage of the ring at 128 x 256 39.9 -> 37.1 us (1024 x 8192 x 4096).
// More stages elsewhere measured nothing; 64 x 128 on four waves 15.4 -> 19.5 us (512 x 4096 x 4096).
template <typename T, int EPI> static int q8(int cfg, const Args& a, hipStream_t s) {
  constexpr int WN64 = EPI == 3 ? 2 : 4;  // gate/up: a wave's columns hold both products
  switch (cfg) {
    case 0: return launch_tile<T, 256, 256, 4, 2, 2, false, false, EPI, false, true>(a, s);
    case 1: return launch_tile<T, 128, 256, 2, 4, 3, false, false, EPI, false, true>(a, s);
    case 2: return launch_tile<T, 128, 128, 2, 4, 4, false, false, EPI, false, true>(a, s);
    case 3: return launch_tile<T, 64, 128, 2, 4, 4, false, false, EPI, false, true>(a, s);
    case 4: return launch_tile<T, 64, 64, WN64 == 2 ? 4 : 2, WN64, 4, false, false, EPI, false, true>(a, s);
    case 6: return launch_tile<T, 192, 256, 4, 2, 2, false, false, EPI, false, true>(a, s);
    case 7: return launch_tile<T, 192, 128, 4, 2, 3, false, false, EPI, false, true>(a, s);
    default: return launch_tile<T, 32, 64, 2, 2, 4, false, false, EPI, false, true>(a, s);
  }
}

int launch_tile_q8(int dtype, int cfg, int epi, const Args& a, hipStream_t s) {
  if (epi == 3) return dtype == Q3_BF16 ? q8<BF16, 3>(cfg, a, s) : q8<F16, 3>(cfg, a, s);
  return dtype == Q3_BF16 ? q8<BF16, 0>(cfg, a, s) : q8<F16, 0>(cfg, a, s);
}

}  // namespace q3gemm
