// What workgroups of one launch tell each other: 8-byte words of two float32, one store each, which
// are their own sign of having been written (unset words hold all ones), so no fence is needed.
// Work that waits is taken by tickets, so that what it waits for already runs or starts next.
#pragma once
#include <stddef.h>

#include "common.h"

namespace ddm {

constexpr uint64_t kUnset = ~0ull;

__device__ __forceinline__ uint64_t word(float a, float b) {
    const uint64_t w = (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a);
    return w == kUnset ? w ^ 1u : w;               // two NaN of all ones: another NaN
}
__device__ __forceinline__ float word_a(uint64_t w) { return __uint_as_float((uint32_t)w); }
__device__ __forceinline__ float word_b(uint64_t w) { return __uint_as_float((uint32_t)(w >> 32)); }
__device__ __forceinline__ void publish(uint64_t* p, uint64_t w) {
    __hip_atomic_store(p, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t peek(const uint64_t* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// A wait gives up after some seconds: a guard against a hang, not a wait.  What was waited for is NaN then, and so
// is what follows from it, and the guard says that it was not the inputs'.  Every source that waits has one.
// The recurrence's waits take the limit as a constant and tell the guard only after the last of them: in the
// wait, either spilled registers (65536 x 2048 bf16 with float32 gates, gradient 570 us instead of 529).
// The distillation's read it, so that a test can set it.
constexpr uint32_t kLooks = 1u << 22;
struct Guard {
    uint32_t looks, gave_up;                   // at most; 1 once a wait took them all
};
[[maybe_unused]] static __device__ Guard guard = {kLooks, 0u};
__device__ __forceinline__ void tell_gave_up() { *(volatile uint32_t*)&guard.gave_up = 1u; }
// The current device's: a new limit (NULL: as it is), and whether a wait gave up since this was last asked (NULL: not
// asked).  After hipDeviceSynchronize.
[[maybe_unused]] static int use_guard(const uint32_t* looks, bool* gave_up) {
    const char* who = "wait guard";
    if (gave_up) {
        const uint32_t none = 0;
        uint32_t one = 0;
        if (int rc = hip_status(hipMemcpyFromSymbol(&one, HIP_SYMBOL(guard), 4, offsetof(Guard, gave_up)), who)) return rc;
        if (one)
            if (int rc = hip_status(hipMemcpyToSymbol(HIP_SYMBOL(guard), &none, 4, offsetof(Guard, gave_up)), who)) return rc;
        *gave_up = *gave_up || one;
    }
    return looks ? hip_status(hipMemcpyToSymbol(HIP_SYMBOL(guard), looks, 4, offsetof(Guard, looks)), who) : 0;
}
int use_guard_distill(const uint32_t* looks, bool* gave_up);
int use_guard_gated(bool* gave_up);
int use_guard_gated_grad(bool* gave_up);
// Queues of tickets: one counter gives out a ticket every 15 ns (measured: 32768 workgroups that took
// one each ran no faster than that), so a launch has up to 8, 256 bytes apart, and a workgroup takes
// from the queue that its index says.  What waits for each other is given out by one queue.
// Workgroups go round the 8 dies, so a queue is eight in a row: every die works for every queue (a queue
// a die: the distillation of 4096 x 131072 took 480 us instead of 442).
constexpr int kQueues = 8, kDies = 8;
// Workgroups for `pieces` pieces of work a queue: as many to every queue.
inline int64_t queue_grid(int64_t pieces, int queues) { return queues * ceil_div(pieces, kDies) * kDies; }
constexpr int64_t kTicketBytes = kQueues * 256;
struct Ticket {
    uint32_t queue, number;     // the same in every lane, and known to be
};
__device__ __forceinline__ Ticket take_ticket(uint32_t* tickets, uint32_t queues) {
    __shared__ uint32_t sh;
    const uint32_t q = blockIdx.x / kDies & (queues - 1u);
    if (threadIdx.x == 0) sh = atomicAdd(tickets + q * 64, 1u);
    __syncthreads();
    return Ticket{q, (uint32_t)__builtin_amdgcn_readfirstlane(sh)};
}

// Before such a launch: tickets 0, words unset; and what is copied on the way (from NULL: zeros).
int reset_words(uint32_t* tickets, uint64_t* words, int64_t nwords, const float* from, float* to, int64_t ncopy,
                hipStream_t stream, const char* who);

}  // namespace ddm
