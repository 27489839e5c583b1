// Resets what words.h's launches wait for.
#include "words.h"

namespace ddm {

__global__ __launch_bounds__(256) void k_reset_words(uint32_t* tickets, uint64_t* words, int64_t nwords,
                                                     const float* from, float* to, int64_t ncopy) {
    const int64_t step = (int64_t)gridDim.x * 256;
    const int64_t i0 = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i0 < kQueues && tickets) tickets[i0 * 64] = 0;
    for (int64_t i = i0; i < nwords; i += step) words[i] = kUnset;
    for (int64_t i = i0; i < ncopy; i += step) to[i] = from ? from[i] : 0.0f;
}

int reset_words(uint32_t* tickets, uint64_t* words, int64_t nwords, const float* from, float* to, int64_t ncopy,
                hipStream_t stream, const char* who) {
    const int64_t most = nwords > ncopy ? nwords : ncopy;
    int64_t grid = ceil_div(most, 256 * 4);
    grid = grid < 1 ? 1 : grid > 2048 ? 2048 : grid;
    k_reset_words<<<dim3((unsigned)grid), 256, 0, stream>>>(tickets, words, nwords, from, to, ncopy);
    return launch_status(who);
}

}  // namespace ddm

extern "C" int ddm_wait_gave_up(int32_t* gave_up) {
    if (!gave_up) {
        ddm::set_error("ddm_wait_gave_up: invalid argument (null pointer)");
        return DDM_E_ARG;
    }
    bool any = false;
    if (int rc = ddm::hip_status(hipDeviceSynchronize(), "ddm_wait_gave_up")) return rc;
    if (int rc = ddm::use_guard_distill(nullptr, &any)) return rc;
    if (int rc = ddm::use_guard_gated(&any)) return rc;
    if (int rc = ddm::use_guard_gated_grad(&any)) return rc;
    *gave_up = any;
    return 0;
}

extern "C" int ddm_wait_limit(uint32_t looks) {
    if (int rc = ddm::hip_status(hipDeviceSynchronize(), "ddm_wait_limit")) return rc;
    return ddm::use_guard_distill(&looks, nullptr);
}
