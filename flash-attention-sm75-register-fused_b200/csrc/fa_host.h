// Host helpers of fa_abi.cu that the paged-cache entry points share.
#pragma once
#include <cuda.h>

namespace fa {

// FA_OK if the current device is an sm_100 part; makes its primary context
// current on the calling thread.
int host_check_device();
int host_sm_count();
// Number of the next watched launch (tags device status words) and the
// watchdog's deadline.
unsigned host_next_epoch();
unsigned long long host_timeout_ns();

// Tiled tensor map of a tensor with the given dimensions, byte strides (of
// dimensions 1 ..; multiples of 16) and box, zero fill, swizzled over the box's
// inner extent (64 or 128 bytes).  Recent encodings are reused.  False if the
// encoder refuses it.
struct TiledMap {
  enum { kF16, kBf16, kBytes };
  const void* base;
  int type, rank;
  unsigned long long dims[5], strides[4];
  unsigned box[5];
};
bool host_tensor_map(CUtensorMap* map, const TiledMap& t);

}  // namespace fa
