// tbh_hostcall.h -- the host-pointer form of an operation: inputs to the
// device's staging buffer, the launches on the device's stream, outputs back,
// one call at a time per device.
#pragma once

#include <initializer_list>
#include <utility>
#include <vector>

#include "tbh_internal.h"

namespace tbh {
namespace {

// Grows the device's staging buffer (callers hold dev->mu).
tbh_status ensure_stage(tbh_device *dev, size_t need) {
    if (dev->stage_bytes >= need) return TBH_OK;
    (void)hipFree(dev->stage);   // replaced below; a failed free leaves nothing to undo
    dev->stage = nullptr;
    dev->stage_bytes = 0;
    hipError_t e = hipMalloc(&dev->stage, need);
    if (e != hipSuccess) return hip_error(e, "staging buffer");
    dev->stage_bytes = need;
    return TBH_OK;
}

size_t pad256(size_t b) { return (b + 255) & ~size_t(255); }

// Host-pointer call: copy the inputs in, run `enqueue` on the device's
// stream, copy the output back, wait.
template <class F>
tbh_status host_call(tbh_device *dev, const char *what, std::initializer_list<std::pair<const void *, size_t>> ins,
                     void *out, size_t out_bytes, F enqueue) {
    std::lock_guard<std::mutex> lock(dev->mu);
    tbh_status st = use_device(dev->ordinal);
    if (st != TBH_OK) return st;
    size_t need = pad256(out_bytes);
    for (auto &in : ins) need += pad256(in.second);
    st = ensure_stage(dev, need);
    if (st != TBH_OK) return st;
    char *p = (char *)dev->stage;
    std::vector<const void *> dptr;
    for (auto &in : ins) {
        if (in.first && in.second) {
            hipError_t e = hipMemcpyAsync(p, in.first, in.second, hipMemcpyHostToDevice, dev->stream);
            if (e != hipSuccess) return hip_error(e, what);
            dptr.push_back(p);
        } else {
            dptr.push_back(nullptr);
        }
        p += pad256(in.second);
    }
    hipError_t e = enqueue(dptr, (void *)p, dev->stream);
    if (e == hipSuccess) e = hipMemcpyAsync(out, p, out_bytes, hipMemcpyDeviceToHost, dev->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(dev->stream);
    if (e != hipSuccess) return hip_error(e, what);
    return TBH_OK;
}

}  // namespace
}  // namespace tbh
