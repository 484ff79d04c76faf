// The product's own 8-bit product and decode kernels with waits that look at the clock at every poll, in a library of the test-suite (not
// part of the product library or its ABI): with a limit of a few cycles their waits run out where the product's would not, so
// that what the kernels do then can be tested.  The waits for a kernel's own copies and products keep their full limit.
#define ESP_MBAR_NEVER_SUSPEND
#define ESP_MBAR_POLLS_PER_LOOK 1u

#include "../../loongserve_b200/csrc/w8a8_gemm.cu"
#include "../../loongserve_b200/csrc/decode_q8.cu"

namespace esp {
char* last_cuda_error_buf() {
    static thread_local char buf[256] = {0};
    return buf;
}
}  // namespace esp

extern "C" int esp_short_limit(int64_t cycles) {
    const int rc = esp::set_mm_wait_limit(cycles);
    return rc ? rc : esp::set_decode_q8_wait_limit(cycles);
}

// the status words of the product and of the decode kernels, and clears them
extern "C" int esp_short_status(int32_t out[8]) {
    ESP_CUDA_TRY(cudaDeviceSynchronize());
    const int rc = esp::mm_w8a8_status(out, 1);
    return rc ? rc : esp::decode_q8_status(out + 4, 1);
}
