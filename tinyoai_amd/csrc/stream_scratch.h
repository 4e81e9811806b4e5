// The scratch of a handle's products on any streams, captured or not: a
// buffer per stream (calls on one stream run in order; the lock keeps one
// call's launches together), one that further streams share in turn, and
// buffers that captured graphs own (scratch.h).
#pragma once

#include <hip/hip_runtime.h>

#include <memory>
#include <mutex>

#include "model.h"
#include "scratch.h"

namespace tinyoai {

// A thread as a user of its hipStreamPerThread. The runtime takes that stream
// away when the thread ends, and from then on neither an event recorded there
// nor a device synchronization waits for what is still running there: two threads that
// enqueued four products each and ended gave wrong sums in 3 of 300 runs, with
// no error. So a thread that has asked for this waits, when it ends and before the
// runtime does that, for the stream on the devices that it asked for.
struct ThreadStream {
  uint64_t number;                 // no other thread's before or after
  std::weak_ptr<const void> life;  // ends with the thread, when its stream is idle
};
ThreadStream thread_stream(int device);

class StreamScratch {
 public:
  ~StreamScratch();
  // launch(scratch) with `bytes` of scratch (null for none) on `st`, which
  // its launches go to. Returns the call's code; may throw std::bad_alloc.
  template <typename Launch>
  int run(hipStream_t st, size_t bytes, const Launch &launch) {
    if (!bytes) {
      const hipError_t e = launch(nullptr);
      return e == hipSuccess ? TINYOAI_OK : hip_fail(e, "product launch");
    }
    std::lock_guard<std::mutex> lock(mu_);
    ScratchPool::Lease lease;
    if (int rc = take(st, bytes, &lease)) return rc;
    hipError_t e = launch(lease.ptr);
    if (lease.shared) {  // also after a launch that failed: an earlier one of the call may run
      const hipError_t r = give_back(st);
      if (e == hipSuccess) e = r;
    }
    return e == hipSuccess ? TINYOAI_OK : hip_fail(e, "product launch");
  }

 private:
  int take(hipStream_t st, size_t bytes, ScratchPool::Lease *lease);
  hipError_t give_back(hipStream_t st);  // the shared buffer, after what `st` holds
  std::mutex mu_;
  ScratchPool pool_;
  hipEvent_t shared_done_ = nullptr;  // after the shared buffer's last call
};

}  // namespace tinyoai
