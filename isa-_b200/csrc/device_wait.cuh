// device_wait.cuh — waits inside kernels that end, and the word that tells the host
// about one that ran out.
//
// A wait that does not end is a lost copy or product: the kernel gives up, lets what
// it has in flight end, hands out NaN and marks the word, and the next call of the
// library's entry points that use such waits fails with that message.  The word is
// host memory that the device sees, so that the host looks at it without waiting.

#ifndef CIMEKV_DEVICE_WAIT_CUH
#define CIMEKV_DEVICE_WAIT_CUH

#include <cstdint>

enum { CIMEKV_WAIT_NORM = 0, CIMEKV_WAIT_PRODUCT = 1, CIMEKV_WAIT_KINDS = 2 };

// The word of `kind` as kernels see it; fails when a wait of any kind has run out since the last
// time that a call said so.
int cimekv_internal_wait_word(int kind, unsigned** word);

__device__ __forceinline__ unsigned long long wall_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

// How long a wait has been on, two seconds at most.  The time between two looks counts for
// 50 ms at most, so that a kernel that was taken off the GPU for longer than the limit (another process's turn, a
// debugger) does not give up on its first look afterwards.
struct Patience {
    unsigned long long last = 0, spent = 0;
    __device__ __forceinline__ bool left(unsigned long long limit = 2000000000ull) {
        const unsigned long long now = wall_ns();
        if (last) spent += now - last < 50000000ull ? now - last : 50000000ull;
        last = now;
        return spent <= limit;
    }
};

// Waits for the phase of `parity` to end.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, unsigned long long limit = 2000000000ull) {
    Patience patience;
    for (int i = 0; i < (1 << 28); ++i) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return true;
        if (!patience.left(limit)) return false;
    }
    return false;
}

__device__ __forceinline__ void mark_lost(unsigned* word) {
    *reinterpret_cast<volatile unsigned*>(word) = 1;
    __threadfence_system();
}

#endif  // CIMEKV_DEVICE_WAIT_CUH
