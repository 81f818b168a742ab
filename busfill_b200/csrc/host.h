// Host-side services that the translation units of the library share: the
// device check, a stream's error words and workspace, and the launch with
// programmatic dependent launch (BUSFILL_OPT_PDL). Defined in busfill.cu.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>

namespace busfill {

// error bit of an out-of-range index in device memory (the kernel roles'
// timeout bits are below it)
constexpr unsigned kErrIndex = 256u;

namespace host {

struct Context {
  int dev = 0;
  int sms = 0;
  unsigned* error = nullptr;   // the stream's device error words
};

// Current device (must be sm_100) and the stream's error words; a busfill_status.
int context(cudaStream_t s, Context* out);

// The workspace of an attention call: the stream's, of `bytes` in every call,
// or, while the stream is capturing, one of `captured_bytes` that belongs to the
// graph. The first `zeroed` bytes are zero when it is made.
int workspace(const Context& c, cudaStream_t s, size_t bytes, size_t captured_bytes, size_t zeroed, void** out);

int launch(const void* kernel, dim3 grid, dim3 block, size_t smem, cudaStream_t s, void** args);

}  // namespace host
}  // namespace busfill
