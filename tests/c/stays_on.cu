// A kernel that lets the next one in its stream start at once and then stays on the GPU for so many milliseconds.  It
// ends by itself: the loop is counted too, at a microsecond or more a turn.
#include <cstdint>
#include <cuda_runtime.h>

__global__ void stays_on(uint64_t ns) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  uint64_t start, now;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(start));
  for (uint32_t turn = 0; turn < 5000000u; ++turn) {
    __nanosleep(1000);
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    if (now - start >= ns) break;
  }
}

extern "C" int launch_stays_on(uint32_t ms, void* stream) {
  stays_on<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(uint64_t(ms) * 1000000u);
  return static_cast<int>(cudaGetLastError());
}
