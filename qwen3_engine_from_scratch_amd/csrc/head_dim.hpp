// The head size that the attention kernels are built for.
#pragma once

namespace {

constexpr int kD = 128;

}  // namespace
