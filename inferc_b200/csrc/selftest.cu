// Self-test of the bounded-wait failure path, without a GPU fault.
//
// Every wait in this library's kernels (mbarrier phases of the TMA /
// tcgen05 pipelines, grid barriers of the persistent decode kernel) gives up
// after a time limit, sets a device error flag and lets its CTA leave; the
// host then reports INFERC_ERR_TIMEOUT from inferc_dev_stream_synchronize and
// the context stays usable. This file runs those wait loops on something that
// is never signalled (an mbarrier nothing arrives at, an arrival counter no
// CTA increments; for a warp's wait an arrival that comes too late for half of
// its lanes) with a caller-chosen short limit, so a test can watch the
// whole path: the wait gives up, the flag is set, the host reads and clears
// it, and later launches work. Nothing here traps, faults or spins without a
// bound.
#include "tc_ptx.cuh"

namespace inferc_dev {
namespace {

__device__ int g_selftest_error;

// One thread waits for an arrival that never comes; then a warp waits for one
// that comes after half of its lanes have run out of time (60 ms later at least)
// and before the others have: the warp has to give up as one.
__global__ void selftest_mbar_kernel(unsigned long long limit_ns) {
  constexpr unsigned long long kLate = 60ull * 1000 * 1000, kLong = 1000ull * 1000 * 1000;
  __shared__ __align__(8) uint64_t never, late;
  if (threadIdx.x == 0) {
    tc::mbar_init(&never, 1);
    tc::mbar_init(&late, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    bool ran_out = true;
    if (threadIdx.x == 0) ran_out = !tc::mbar_wait(&never, 0, limit_ns);
    __syncwarp();
    const bool done = tc::warp_wait(&late, 0, threadIdx.x < 16 ? limit_ns : limit_ns + kLong);
    const bool none = __ballot_sync(0xffffffffu, done) == 0;
    if (threadIdx.x == 0 && ran_out && none) atomicExch(&g_selftest_error, 1);
  } else if (threadIdx.x == 32) {
    const unsigned long long t0 = tc::gclock_ns();
    while (tc::gclock_ns() - t0 < 2 * limit_ns + kLate) __nanosleep(10000);
    tc::mbar_arrive(&late);
  }
  __syncthreads();
}

// The grid-barrier wait of the persistent decode kernel: thread 0 polls an
// arrival counter with acquire loads until it reaches its target, giving up
// after limit_ns (checked every 64 polls) or when another CTA flagged an error.
__global__ void selftest_grid_kernel(unsigned int* counter, unsigned long long limit_ns) {
  if (threadIdx.x == 0) {
    const unsigned target = gridDim.x + 1;  // one more arrival than CTAs exist
    atomicAdd(counter, 1u);
    const unsigned long long t0 = tc::gclock_ns();
    for (uint32_t i = 0;;) {
      unsigned v;
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(counter) : "memory");
      if ((int)(v - target) >= 0) break;
      if ((++i & 63) == 0 &&
          (tc::gclock_ns() - t0 > limit_ns || *(volatile int*)&g_selftest_error)) {
        atomicExch(&g_selftest_error, 1);
        break;
      }
    }
  }
  __syncthreads();
}

}  // namespace

int read_and_clear_selftest_error() {
  int v = 0;
  IDEV_CUDA(cudaMemcpyFromSymbol(&v, g_selftest_error, sizeof(int)));
  if (v) {
    const int z = 0;
    IDEV_CUDA(cudaMemcpyToSymbol(g_selftest_error, &z, sizeof(int)));
  }
  return v;
}

}  // namespace inferc_dev

extern "C" int inferc_dev_selftest_wait_timeout(int which, int64_t limit_us, void* stream) {
  using namespace inferc_dev;
  return guard([&] {
    IDEV_CHECK_ARG(which == 0 || which == 1, "selftest: which must be 0 (mbarrier) or 1 (grid)");
    IDEV_CHECK_ARG(limit_us >= 1 && limit_us <= 1000000, "selftest: limit must be in [1us, 1s]");
    cudaStream_t st = as_stream(stream);
    const unsigned long long ns = (unsigned long long)limit_us * 1000ull;
    if (which == 0) {
      selftest_mbar_kernel<<<1, 64, 0, st>>>(ns);
      IDEV_LAUNCHED();
    } else {
      void* counter = nullptr;
      IDEV_CUDA(cudaMallocAsync(&counter, sizeof(unsigned int), st));
      IDEV_CUDA(cudaMemsetAsync(counter, 0, sizeof(unsigned int), st));
      selftest_grid_kernel<<<4, 32, 0, st>>>(static_cast<unsigned int*>(counter), ns);
      IDEV_LAUNCHED();
      IDEV_CUDA(cudaFreeAsync(counter, st));
    }
  });
}
