// What the segments of a scan leave if nothing enters them, and their decays (ScanArgs::ends): of the states from the front, or of their gradients from the back.
#pragma once
#include "state_space.cuh"

namespace hdla {

template <typename T> hipError_t launch_scan_ends(const ScanArgs& a, const ScanPlan& s, bool back, hipStream_t stream);

}  // namespace hdla
