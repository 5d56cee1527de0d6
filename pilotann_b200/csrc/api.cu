// Error plumbing and bookkeeping shared by the C-ABI entry points.
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <mutex>

#include "pa_common.cuh"

namespace pa {

static thread_local char g_error[512] = "";
static std::atomic<int64_t> g_launches{0};

int fail(int code, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_error, sizeof g_error, fmt, ap);
    va_end(ap);
    return code;
}

int cuda_fail(cudaError_t err, const char *what) {
    snprintf(g_error, sizeof g_error, "%s: %s (%d)", what, cudaGetErrorString(err),
             static_cast<int>(err));
    return PA_ERR_CUDA;
}

// Whether a grouped or 4-bit product gave up on a wait, a word for each device: in host memory that the
// kernels write to, so that the next call sees it without waiting for the GPU.
constexpr int kDevices = 64;
static std::atomic<int *> g_gave_up{nullptr};

int *product_status_address() {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kDevices) return nullptr;
    int *words = g_gave_up.load(std::memory_order_acquire);
    if (words == nullptr) {
        static std::mutex once;
        std::lock_guard<std::mutex> lock(once);
        words = g_gave_up.load(std::memory_order_acquire);
        if (words == nullptr) {
            // the first call may be one that is captured into a graph
            cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
            if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) return nullptr;
            void *p = nullptr;
            const cudaError_t rc = cudaHostAlloc(&p, kDevices * sizeof(int),
                                                 cudaHostAllocPortable | cudaHostAllocMapped);
            (void)cudaThreadExchangeStreamCaptureMode(&mode);
            if (rc != cudaSuccess) {
                (void)cudaGetLastError();
                return nullptr;
            }
            words = static_cast<int *>(p);
            for (int i = 0; i < kDevices; ++i) words[i] = 0;
            g_gave_up.store(words, std::memory_order_release);
        }
    }
    return words + dev;  // unified addressing: the same on the device
}

int product_status(bool reset) {
    int dev = 0;
    volatile int *words = g_gave_up.load(std::memory_order_acquire);
    if (words == nullptr || cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kDevices) return 0;
    const int status = words[dev];
    if (reset) words[dev] = 0;
    return status;
}

int product_check() {
    if (product_status(false) == 0) return PA_OK;
    return fail(PA_ERR_CUDA, "a grouped or 4-bit product gave up on a wait; its result is NaN "
                             "(pa_device_status(1) clears this)");
}

void count_launch(int n) { g_launches.fetch_add(n, std::memory_order_relaxed); }

}  // namespace pa

// 106: long sums in parts, products that give up are NaN and seen by the next call
extern "C" int pa_version(void) { return 106; }
extern "C" const char *pa_last_error(void) { return pa::g_error; }
extern "C" int64_t pa_launch_count(void) { return pa::g_launches.load(std::memory_order_relaxed); }
