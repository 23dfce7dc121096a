// Library-wide pieces of the C ABI: version, per-thread error text, the
// device flag word and the per-device SM count cache.
#include <atomic>
#include <mutex>
#include <string>
#include <vector>

#include "cx_common.cuh"  // unity build: included from cxkv.cu

namespace cx {

static thread_local std::string t_last_error;

void set_error(const std::string& msg) { t_last_error = msg; }

int fail(int code, const std::string& msg) {
    t_last_error = msg;
    return code;
}

int cuda_fail(cudaError_t e, const char* what) {
    t_last_error = std::string(what) + ": " + cudaGetErrorString(e);
    return CX_ERR_CUDA;
}

int num_sms() {
    static std::mutex mu;
    static std::vector<int> cache;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    std::lock_guard<std::mutex> lk(mu);
    if ((int)cache.size() <= dev) cache.resize(dev + 1, 0);
    if (cache[dev] == 0) {
        int n = 0;
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
        cache[dev] = n;
    }
    return cache[dev];
}

// The flag words of all translation units, collected (and cleared) by one launch into
// the word of a call (of the last kFlagCalls): one copy to the host.  A copy a unit took
// 47 us a call with four units (27 with two).
constexpr unsigned int kFlagCalls = 64;
static __device__ unsigned int g_all_flags[kFlagCalls];
struct FlagWords {
    unsigned int* w[4];
};
static __global__ void collect_flags_kernel(const FlagWords words, int clear, unsigned int* to) {
    unsigned int v = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) v |= clear ? atomicExch(words.w[i], 0u) : atomicOr(words.w[i], 0u);
    *to = v;
}

}  // namespace cx

extern "C" {

const char* cx_version(void) { return "cxkv 0.1 sm_100a"; }

const char* cx_last_error(void) { return cx::t_last_error.c_str(); }

int cx_device_error(void* stream, int clear, uint32_t* flags) {
    if (!flags) return cx::fail(CX_ERR_SHAPE, "cx_device_error: flags is NULL");
    cudaStream_t s = cx::as_stream(stream);
    const cx::FlagWords words{{cx::dev_flags(), cx::dev_flags_scored(), cx::dev_flags_tree(),
                               cx::dev_flags_latent()}};
    void* all = nullptr;
    CX_CUDA_CHECK(cudaGetSymbolAddress(&all, cx::g_all_flags));
    for (unsigned int* w : words.w)
        if (!w) return cx::fail(CX_ERR_CUDA, "cx_device_error: no flag word on this device");
    static std::atomic<unsigned int> calls{0};
    unsigned int* to = static_cast<unsigned int*>(all) + calls++ % cx::kFlagCalls;
    cx::collect_flags_kernel<<<1, 1, 0, s>>>(words, clear, to);
    const int rc = cx::check_launch("collect_flags_kernel");
    if (rc) return rc;
    unsigned int v = 0;
    CX_CUDA_CHECK(cudaMemcpyAsync(&v, to, sizeof(v), cudaMemcpyDeviceToHost, s));
    CX_CUDA_CHECK(cudaStreamSynchronize(s));
    *flags = v;
    return CX_OK;
}

}  // extern "C"
