// Error text, ABI version and the per-device scratch arena.
#include "common.h"

#include <map>
#include <mutex>
#include <tuple>

namespace evfly {

std::string &last_error_ref() {
    static thread_local std::string s;
    return s;
}

int fail(int code, const char *fmt, ...) {
    char buf[1024];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    last_error_ref() = buf;
    return code;
}

namespace {
struct Scratch {
    void *ptr = nullptr;
    size_t cap = 0;
};
std::map<std::tuple<int, hipStream_t, int>, Scratch> g_scratch;   // (device, stream, slot)
std::mutex g_scratch_mu;
}  // namespace

int scratch_get(size_t bytes, void **out, hipStream_t stream, int slot) {
    int dev = 0;
    EVFLY_HIP(hipGetDevice(&dev));
    std::lock_guard<std::mutex> lk(g_scratch_mu);
    Scratch &s = g_scratch[std::make_tuple(dev, stream, slot)];
    if (s.cap < bytes) {
        if (s.ptr) EVFLY_HIP(hipFree(s.ptr));
        s.ptr = nullptr;
        s.cap = 0;
        size_t want = bytes + (bytes >> 2) + (1 << 20);
        EVFLY_HIP(hipMalloc(&s.ptr, want));
        s.cap = want;
    }
    *out = s.ptr;
    return 0;
}

namespace {
// bytes up to the first 16-byte boundary and behind the last one singly, the rest in 16-byte pieces
__global__ __launch_bounds__(256) void k_fill_bytes(unsigned char *dst, unsigned word, size_t head, size_t pieces, size_t tail) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i < head) dst[i] = (unsigned char)word;
    if (i < tail) dst[head + pieces * 16 + i] = (unsigned char)word;
    for (size_t k = i; k < pieces; k += (size_t)gridDim.x * 256) reinterpret_cast<uint4 *>(dst + head)[k] = make_uint4(word, word, word, word);
}
}  // namespace

int fill_bytes(void *dst, unsigned char value, size_t bytes, hipStream_t stream) {
    if (bytes == 0) return 0;
    size_t head = (16 - (reinterpret_cast<uintptr_t>(dst) & 15)) & 15;
    if (head > bytes) head = bytes;
    const size_t pieces = (bytes - head) / 16, tail = bytes - head - pieces * 16;
    const size_t need = (pieces + 255) / 256, most = 8 * kNumCU;
    hipLaunchKernelGGL(k_fill_bytes, dim3((unsigned)(need < 1 ? 1 : need < most ? need : most)), dim3(256), 0, stream, static_cast<unsigned char *>(dst), value * 0x01010101u,
                       head, pieces, tail);
    EVFLY_LAUNCH_CHECK();
    return 0;
}

}  // namespace evfly

extern "C" int evfly_abi_version(void) { return EVFLY_ABI_VERSION; }
extern "C" const char *evfly_last_error(void) { return evfly::last_error_ref().c_str(); }
