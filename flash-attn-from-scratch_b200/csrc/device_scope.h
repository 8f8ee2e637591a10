// device_scope.h — the device that a call of this library runs on.
//
// The library shares its thread's current context with its caller (torch, or any other user of
// CUDA in the process), and either may change it between two calls: what this library made current
// once says nothing about now, so every call asks.  A call that has to switch puts the caller's
// context back when it ends -- the context, not a device number: to set a device is to create a
// context on it, and a thread that had none is to have none again.  Device 0 is the exception: it is
// where a thread without a context is anyway, so its context may stay (torch's autograd threads begin
// so, and warn if they find none).
//
// Host code without CUDA in it, so that a test can run it against a stand-in.  Api is that of the
// driver and runtime; its functions return 0 or an error:
//   current_device(int*)    the current context's device; an error where there is none
//   current_context(void**) nullptr where there is none
//   set_context(void*)
//   set_device(int)         makes the device's primary context current
#pragma once

namespace lk {

// What a thread remembers between calls.
struct ThreadDevice {
  int device = -1;  // picked with lk_set_device, or that of the last call with a stream of its own
  int seen = -1;    // the caller's current device at that time (-1: it had no context)

  // Calls on the legacy default stream, which names no device.
  int for_null_stream() const { return device >= 0 ? device : 0; }
  // Calls that name no stream (the status word, ...): the device of the thread's last call, or the
  // current one (`now`, -1: none) where the caller has changed it since.
  int for_status(int now) const { return now >= 0 && (device < 0 || now != seen) ? now : for_null_stream(); }
};

template <class Api>
class DeviceSwitch {
 public:
  DeviceSwitch() = default;
  DeviceSwitch(const DeviceSwitch&) = delete;
  ~DeviceSwitch() {
    if (restore_) Api::set_context(before_);
  }
  // The caller's current device, -1 where it has none.
  static int now() {
    int dev = -1;
    return Api::current_device(&dev) == 0 ? dev : -1;
  }
  // Makes `dev` current until this object goes; `t` remembers it.  At most once per object, and one
  // object at a time on a thread.
  int to(int dev, ThreadDevice& t) {
    const int was = now();
    if (was != dev) {
      // A context that is current but answers for no device has been destroyed: not put back.
      restore_ = Api::current_context(&before_) == 0 && (was >= 0 || (before_ == nullptr && dev != 0));
      if (const int st = Api::set_device(dev)) return st;
    }
    t.device = dev;
    t.seen = was;
    return 0;
  }

 private:
  void* before_ = nullptr;
  bool restore_ = false;
};

}  // namespace lk
