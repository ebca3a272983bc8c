// Two host threads ask for different amounts of shared memory for one kernel at the same time, against stand-ins for the
// two runtime calls that hold the first setter until the second has set its own.  Afterwards both sizes must be allowed.
#include <condition_variable>
#include <cstdio>
#include <mutex>
#include <thread>

#include "fv_common.h"

static std::mutex m;
static std::condition_variable cv;
static int inside = 0;
static int limit = 48 << 10;

extern "C" cudaError_t cudaGetDevice(int* d) {
  *d = 0;
  return cudaSuccess;
}
extern "C" cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int value) {
  std::unique_lock<std::mutex> l(m);
  limit = value;
  ++inside;
  cv.notify_all();
  cv.wait_for(l, std::chrono::milliseconds(500), [] { return inside == 2; });
  return cudaSuccess;
}

int main() {
  static std::atomic<bool> given[64];
  const int kernel = 0;
  const size_t wide = 100 << 10, less = 60 << 10, most = 208 << 10;
  std::thread a([&] { fv::allow_smem(&kernel, given, wide, most); });
  {  // the wide one sets first
    std::unique_lock<std::mutex> l(m);
    cv.wait(l, [] { return inside == 1; });
  }
  std::thread b([&] { fv::allow_smem(&kernel, given, less, most); });
  a.join();
  b.join();
  for (size_t need : {wide, less, most})
    if (fv::allow_smem(&kernel, given, need, most) != cudaSuccess || (size_t)limit < need) {
      std::printf("%zu bytes asked for, %d allowed\n", need, limit);
      return 1;
    }
  return fv::allow_smem(&kernel, given, most + 1, most) == cudaErrorInvalidValue ? 0 : 1;
}
