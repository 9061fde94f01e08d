// Host-side state shared by the libraries' entry points: the calling thread's error text, launch facts
// per device. Linked into each library, so each has an error text of its own.
#include <map>
#include <mutex>
#include <string>
#include <tuple>

#include "w4a8_internal.h"

namespace w4a8 {

namespace {
thread_local std::string g_error;
}

const std::string& last_error() { return g_error; }

void set_error(const std::string& msg) { g_error = msg; }

KernelStamp& next_kernel_stamp() {
    thread_local KernelStamp stamp;
    return stamp;
}
void clear_error() { g_error.clear(); }

int check_launch(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        set_error(std::string(what) + ": " + hipGetErrorString(e));
        return W4A8_ERR_HIP;
    }
    return W4A8_OK;
}

namespace {
std::mutex g_dev_mu;
// (device, kind, kernel, threads, lds) -> cached value; kind 0: LDS reserved, 1: blocks
// per CU, 2: CU count
std::map<std::tuple<int, int, const void*, int, size_t>, int> g_dev_facts;
int current_device() {
    int dev = 0;
    return hipGetDevice(&dev) == hipSuccess ? dev : 0;
}
}  // namespace

int reserve_dyn_lds(const void* kernel, int bytes, const char* what) {
    const auto key = std::make_tuple(current_device(), 0, kernel, 0, (size_t)bytes);
    std::lock_guard<std::mutex> lock(g_dev_mu);
    if (g_dev_facts.count(key)) return W4A8_OK;
    const hipError_t e =
        hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) {
        set_error(std::string(what) + ": cannot reserve dynamic LDS: " + hipGetErrorString(e));
        return W4A8_ERR_HIP;
    }
    g_dev_facts[key] = 1;
    return W4A8_OK;
}

int device_cu_count() {
    const int dev = current_device();
    const auto key = std::make_tuple(dev, 2, (const void*)nullptr, 0, (size_t)0);
    std::lock_guard<std::mutex> lock(g_dev_mu);
    auto it = g_dev_facts.find(key);
    if (it != g_dev_facts.end()) return it->second;
    int ncu = 0;
    if (hipDeviceGetAttribute(&ncu, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
        ncu <= 0)
        ncu = 256;
    g_dev_facts[key] = ncu;
    return ncu;
}

int blocks_per_cu(const void* kernel, int threads, size_t lds) {
    const auto key = std::make_tuple(current_device(), 1, kernel, threads, lds);
    std::lock_guard<std::mutex> lock(g_dev_mu);
    auto it = g_dev_facts.find(key);
    if (it != g_dev_facts.end()) return it->second;
    int occ = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&occ, kernel, threads, lds) != hipSuccess ||
        occ < 0)
        occ = 0;
    g_dev_facts[key] = occ;
    return occ;
}

}  // namespace w4a8
