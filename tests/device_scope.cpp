// Runs csrc/device_scope.h against a stand-in for CUDA: a thread's current context, which both the
// "library" and the "caller" change.  Prints what failed; exits 0 if nothing did.
#include "device_scope.h"

#include <cstdio>
#include <initializer_list>

namespace {

int g_failed = 0;
#define CHECK(x)                                        \
  do {                                                  \
    if (!(x)) {                                         \
      std::printf("line %d: %s\n", __LINE__, #x);       \
      ++g_failed;                                       \
    }                                                   \
  } while (0)

struct Context {
  int device;
  bool alive;
};
Context g_primary[2] = {{0, false}, {1, false}};
Context* g_current = nullptr;
int g_sets = 0;
bool g_fail = false;

struct Fake {
  static int current_device(int* dev) {
    if (!g_current || !g_current->alive) return 201;
    *dev = g_current->device;
    return 0;
  }
  static int current_context(void** c) {
    *c = g_current;
    return 0;
  }
  static int set_context(void* c) {
    g_current = static_cast<Context*>(c);
    return 0;
  }
  static int set_device(int dev) {
    if (g_fail) return 46;
    ++g_sets;
    g_primary[dev].alive = true;
    g_current = &g_primary[dev];
    return 0;
  }
};

int current() { return lk::DeviceSwitch<Fake>::now(); }

// A call of the library: returns the device that its kernel would be launched on.
int call(lk::ThreadDevice& t, int dev) {
  lk::DeviceSwitch<Fake> s;
  if (s.to(dev, t)) return -2;
  return current();
}

void start(int device) {
  g_primary[0].alive = g_primary[1].alive = false;
  g_current = nullptr;
  if (device >= 0) Fake::set_device(device);
  g_sets = 0;
}

}  // namespace

int main() {
  {  // The caller switches to device 1, calls, switches back, and calls with device 1's tensors again.
    lk::ThreadDevice t;
    start(0);
    Fake::set_device(1);
    CHECK(call(t, 1) == 1 && current() == 1);
    Fake::set_device(0);
    CHECK(t.for_null_stream() == 1);
    CHECK(call(t, t.for_null_stream()) == 1);
    CHECK(current() == 0);
  }
  {  // Either device after the other; the caller's stays.
    lk::ThreadDevice t;
    start(0);
    for (int dev : {1, 0, 1, 1, 0}) CHECK(call(t, dev) == dev && current() == 0 && t.device == dev);
  }
  {  // Nothing is set where the device is current already.
    lk::ThreadDevice t;
    start(0);
    CHECK(call(t, 0) == 0 && g_sets == 0);
  }
  {  // A thread without a context has none afterwards, and no other device gets one.
    lk::ThreadDevice t;
    start(-1);
    CHECK(call(t, 1) == 1 && g_current == nullptr && !g_primary[0].alive);
    CHECK(call(t, 1) == 1 && g_current == nullptr);
    CHECK(call(t, 0) == 0 && current() == 0);  // but device 0 is where such a thread is
    CHECK(call(t, 1) == 1 && current() == 0);
  }
  {  // A device that cannot be set: the error, and the caller's context.
    lk::ThreadDevice t;
    start(0);
    g_fail = true;
    CHECK(call(t, 1) == -2 && current() == 0 && t.device == -1);
    g_fail = false;
  }
  {  // A destroyed context is not put back.
    lk::ThreadDevice t;
    start(0);
    g_primary[0].alive = false;
    CHECK(call(t, 1) == 1 && current() == 1);
  }
  {  // The status word's device: the last call's, or the one that the caller has switched to since.
    lk::ThreadDevice t;
    CHECK(t.for_status(-1) == 0 && t.for_status(1) == 1);
    start(0);
    call(t, 1);
    CHECK(t.for_status(current()) == 1);
    Fake::set_device(1);
    call(t, 1);
    Fake::set_device(0);
    CHECK(t.for_status(current()) == 0);
    start(-1);
    call(t, 1);
    CHECK(t.for_status(current()) == 1);
  }
  return g_failed ? 1 : 0;
}
