// Decode kernel instantiations behind a window, contiguous caches: 2-bit keys and values.
#include "pqkv_decode_mfma.h"

namespace pqkv {

hipError_t launch_dm_window_k2v2(const DecodeArgs &a, hipStream_t s) {
  return launch_dm_widths<2, 2, false, false, false, true>(a, s);
}

}  // namespace pqkv
