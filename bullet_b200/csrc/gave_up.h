// The word by which a device's dense kernels tell the host that a wait of theirs gave up (Waits in tensor.cuh).
#pragma once

namespace b200 {

// For kernels of `device` and the host alike, or null where the device cannot share memory while it is running.
int* gave_up_word(int device);
// Whether it is set; it is 0 then.
bool take_gave_up(int* word);

}  // namespace b200
