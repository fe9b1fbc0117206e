// Shared by the translation units of libroller_hip.so, not part of its interface.
#ifndef ROLLER_INTERNAL_H
#define ROLLER_INTERNAL_H

#include <hip/hip_runtime_api.h>

#include <mutex>

#define RL_HIDDEN __attribute__((visibility("hidden")))

// Error text of the calling thread (rl_last_error); returns `code`.
RL_HIDDEN int rl_fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
// Status of a HIP call that failed, with text.
RL_HIDDEN int rl_hip_fail(hipError_t e, const char* what);
// The device of rl_init and its compute units; RL_ERR_NO_DEVICE (with text) before rl_init.
RL_HIDDEN int rl_device(int* device, int* compute_units);
// Frees what the products keep for a stream that is about to be destroyed.
RL_HIDDEN int rl_products_forget_stream(hipStream_t stream);

// Makes the device of rl_init the calling thread's for a call and puts the caller's back afterwards.
class DeviceScope {
 public:
  DeviceScope() {
    status_ = rl_device(&device_, &compute_units_);
    if (status_) return;
    hipError_t e = hipGetDevice(&before_);
    if (e == hipSuccess && before_ != device_) {
      e = hipSetDevice(device_);
      changed_ = e == hipSuccess;
    }
    if (e != hipSuccess) status_ = rl_hip_fail(e, "selecting the device");
  }
  ~DeviceScope() {
    if (changed_) (void)hipSetDevice(before_);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
  int status() const { return status_; }
  int device() const { return device_; }
  int compute_units() const { return compute_units_; }

 private:
  int status_ = 0, device_ = -1, before_ = -1, compute_units_ = 0;
  bool changed_ = false;
};

// Workspace of one product call: the caller's, or the library's for the stream (one per stream, grown on
// demand, held locked until the call has enqueued everything).  The library's is refused while the stream
// is being captured (the graph would keep an address that a later call may free or share) and for
// hipStreamPerThread (one handle, another stream in every thread).
class ProductRoom {
 public:
  // Takes `need` bytes (rounded up to 256 by the caller); *out may be NULL when need is 0.
  int take(hipStream_t stream, void* user, size_t user_bytes, size_t need, const char* what, char** out);

 private:
  std::unique_lock<std::mutex> lock_;
};

#endif
