// device_wait.cu — the host's side of waits that run out (see device_wait.cuh).

#include <cuda_runtime.h>

#include <atomic>
#include <cstdio>
#include <mutex>

#include "cimekv.h"
#include "device_wait.cuh"

int cimekv_internal_begin_call();
int cimekv_internal_no_pending_error();
void cimekv_internal_set_error(const char* msg);

namespace {

// A page of its own, pinned and made visible to all devices at the first call: the library
// allocates nothing.
alignas(4096) std::atomic<unsigned> g_words[4096 / sizeof(std::atomic<unsigned>)];
static_assert(sizeof(std::atomic<unsigned>) == sizeof(unsigned), "kernels write the words as they are");

int fail(int code, const char* msg) {
    cimekv_internal_set_error(msg);
    return code;
}

int words(unsigned** device) {
    static std::mutex mutex;
    static std::atomic<bool> pinned{false};
    if (!pinned.load(std::memory_order_acquire)) {
        std::lock_guard<std::mutex> lock(mutex);
        if (!pinned.load(std::memory_order_relaxed)) {
            cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;  // the page is not part of anybody's capture
            (void)cudaThreadExchangeStreamCaptureMode(&mode);
            const cudaError_t e = cudaHostRegister(g_words, sizeof(g_words), cudaHostRegisterPortable | cudaHostRegisterMapped);
            (void)cudaThreadExchangeStreamCaptureMode(&mode);
            if (e != cudaSuccess) {
                (void)cudaGetLastError();
                return fail(CIMEKV_ECUDA, cudaGetErrorString(e));
            }
            pinned.store(true, std::memory_order_release);
        }
    }
    static std::atomic<void*> seen[64];  // where each device sees the page
    int dev;
    if (cudaGetDevice(&dev) != cudaSuccess) return fail(CIMEKV_ECUDA, "no current device");
    void* at = dev < 64 ? seen[dev].load(std::memory_order_acquire) : nullptr;
    if (!at) {
        if (cudaHostGetDevicePointer(&at, g_words, 0) != cudaSuccess) {
            (void)cudaGetLastError();
            return fail(CIMEKV_ECUDA, "the words of lost waits are not visible to this device");
        }
        if (dev < 64) seen[dev].store(at, std::memory_order_release);
    }
    *device = static_cast<unsigned*>(at);
    return CIMEKV_OK;
}

__global__ void wait_probe_kernel(unsigned* word, unsigned long long limit) {
    __shared__ __align__(8) uint64_t bar;
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(&bar);
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(at) : "memory");
    if (!mbar_wait(at, 0, limit)) mark_lost(word);  // nothing arrives there
}

}  // namespace

int cimekv_internal_wait_word(int kind, unsigned** word) {
    unsigned* at;
    if (int rc = words(&at)) return rc;
    bool lost = false;
    for (int k = 0; k < CIMEKV_WAIT_KINDS; ++k)
        if (g_words[k].load(std::memory_order_relaxed) && g_words[k].exchange(0)) lost = true;
    if (lost)
        return fail(CIMEKV_ELOST, "a wait in an earlier launch ran out: what that launch was to write is NaN (this call "
                                  "has not been carried out)");
    *word = at + kind;
    return CIMEKV_OK;
}

extern "C" unsigned int cimekv_lost_waits(int reset) {
    unsigned int kinds = 0;
    for (int k = 0; k < CIMEKV_WAIT_KINDS; ++k)
        if (reset ? g_words[k].exchange(0) : g_words[k].load()) kinds |= 1u << k;
    return kinds;
}

extern "C" int cimekv_debug_lose_wait(int kind, float milliseconds, void* stream) {
    int rc = cimekv_internal_begin_call();
    if (rc) return rc;
    if (kind < 0 || kind >= CIMEKV_WAIT_KINDS || !(milliseconds > 0.0f && milliseconds <= 1000.0f))
        return fail(CIMEKV_EINVAL_SHAPE, "debug wait: kind 0 or 1, up to 1000 milliseconds");
    unsigned* at;
    if ((rc = words(&at)) || (rc = cimekv_internal_no_pending_error())) return rc;
    wait_probe_kernel<<<1, 1, 0, (cudaStream_t)stream>>>(at + kind, (unsigned long long)(1e6f * milliseconds));
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? CIMEKV_OK : fail(CIMEKV_ECUDA, cudaGetErrorString(e));
}
