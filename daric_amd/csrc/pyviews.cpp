// daric_tensor views of Python tensor objects, for the ctypes binding.
//
// A tensor's address, shape, strides, type and device read attribute by attribute in
// Python take 1 us on the host, eight of a call 7.6 us: twice as long as the launch. torch
// hands out a C function that reads them from the object (the "dlpack_exchange_api"
// capsule of its tensor class); this entry point calls it. It needs no Python or
// torch header: the objects are passed on as pointers, and the caller holds the
// interpreter's lock (ctypes.PyDLL), so an exception the function sets is raised there.
#include <cstring>

#include "../../include/daric_cache_ops.h"

namespace {

// DLPack's DLTensor, a public C ABI.
struct DlTensor {
    void* data;
    int32_t device_type, device_id;
    int32_t ndim;
    uint8_t code, bits;
    uint16_t lanes;
    int64_t* shape;
    int64_t* strides;
    uint64_t byte_offset;
};
static_assert(sizeof(DlTensor) == 48, "DLTensor layout");
using FromObject = int (*)(void* object, DlTensor* out);

constexpr int32_t kDlCuda = 2, kDlRocm = 10;

int dtype_of(uint8_t code, uint8_t bits) {
    switch (code << 8 | bits) {
        case 0 << 8 | 32: return DARIC_DTYPE_INT32;
        case 0 << 8 | 64: return DARIC_DTYPE_INT64;
        case 1 << 8 | 8: return DARIC_DTYPE_UINT8;
        case 2 << 8 | 16: return DARIC_DTYPE_FLOAT16;
        case 2 << 8 | 32: return DARIC_DTYPE_FLOAT32;
        case 4 << 8 | 16: return DARIC_DTYPE_BFLOAT16;
        case 10 << 8 | 8: return DARIC_DTYPE_FP8_E4M3FN;
        default: return DARIC_DTYPE_OTHER;
    }
}

int view(FromObject from, void* object, daric_tensor* out) {
    DlTensor d;
    if (from(object, &d) != 0) return 1;
    if (d.ndim < 0 || d.ndim > DARIC_MAX_DIMS || (d.ndim > 0 && d.strides == nullptr)) return 2;
    out->data = d.data == nullptr ? nullptr : static_cast<uint8_t*>(d.data) + d.byte_offset;
    out->ndim = d.ndim;
    out->elem_size = d.bits * d.lanes / 8;
    out->device = d.device_type == kDlRocm || d.device_type == kDlCuda ? d.device_id : -1;
    out->dtype = d.lanes == 1 ? dtype_of(d.code, d.bits) : DARIC_DTYPE_OTHER;
    std::memcpy(out->sizes, d.shape, sizeof(int64_t) * d.ndim);
    std::memcpy(out->strides, d.strides, sizeof(int64_t) * d.ndim);
    return 0;
}

}  // namespace

extern "C" {

// The views of n objects; those that are `none` are left as they are. 1: `from` failed (and
// has set an exception), 2: a rank that has no view.
int daric_py_views(void* from, void* none, daric_tensor* out, int n, void* const* objects) {
    for (int i = 0; i < n; ++i) {
        if (objects[i] == none) continue;
        const int status = view(reinterpret_cast<FromObject>(from), objects[i], out + i);
        if (status != 0) return status;
    }
    return 0;
}

}  // extern "C"
