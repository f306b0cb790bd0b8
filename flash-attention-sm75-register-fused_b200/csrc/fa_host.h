// Host helpers of fa_abi.cu that the paged-cache entry points share.
#pragma once

namespace fa {

// FA_OK if the current device is an sm_100 part; makes its primary context
// current on the calling thread.
int host_check_device();
int host_sm_count();

}  // namespace fa
