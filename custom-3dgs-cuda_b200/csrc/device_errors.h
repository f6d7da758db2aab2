// Bits of the device error word (gs_device_error_bits).
#pragma once

namespace gs {

// Device error bits (OR-ed into g_device_errors by the kernels).
constexpr unsigned kErrLookbackTimeout = 1u;  // a decoupled look-back wait hit its limit
constexpr unsigned kErrCapacity = 2u;         // pair count exceeded the pair capacity
constexpr unsigned kErrBadIndex = 4u;         // an index was out of range
constexpr unsigned kErrPeerTimeout = 8u;      // a cross-GPU barrier wait hit its limit
constexpr unsigned kErrCopyTimeout = 16u;     // a wait for a tensor-memory-accelerator copy hit its limit
constexpr unsigned kErrMmaTimeout = 32u;      // a wait inside an attention kernel hit its limit

}  // namespace gs
