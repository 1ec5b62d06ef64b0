// Status words of the serving library's kernels with bounded waits (0: none gave up).
#pragma once

namespace cb200 {

int prefix_device_status(bool reset);
int logprobs_device_status(bool reset);

}  // namespace cb200
