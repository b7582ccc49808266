// igs_feature_host.h -- host side shared by the units of the feature operators: argument checks, the
// device's size.  Included inside their anonymous namespaces.
#pragma once

constexpr int64_t kMaxCount = 0x7FFFFFFE;
constexpr int kMaxRow = 1 << 20;

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t at_most(int64_t v, int64_t most) { return v < most ? v : most; }

// From so many bytes on a tensor is read or written past the caches: three quarters of the last-level cache.
constexpr int64_t kStreamBytes = 192ll << 20;

inline int launch_status() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? IGS_OK : (int)e;
}

inline bool dtype_ok(int t) { return t == IGS_F32 || t == IGS_F16 || t == IGS_BF16; }
inline int dtype_bytes(int t) { return t == IGS_F32 ? 4 : 2; }
inline bool aligned_to(const void* p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

int make_dropout(int threshold, uint64_t seed, const uint64_t* seed_device, uint64_t offset, Dropout* d) {
    if (threshold < 0 || threshold > 65536) return IGS_ERR_BAD_ARGUMENT;
    if (!aligned_to(seed_device, 8)) return IGS_ERR_ALIGNMENT;
    d->threshold = (uint32_t)threshold;
    d->factor = threshold < 65536 ? (float)(65536.0 / (65536 - threshold)) : 0.0f;
    d->seed = seed;
    d->offset = offset;
    d->seed_device = seed_device;
    return IGS_OK;
}

// Compute units of the current device (of an MI355X where there is none: plans are made without a GPU too).
int device_cus() {
    static std::atomic<int> cached{0};
    int cus = cached.load(std::memory_order_relaxed);
    if (cus > 0) return cus;
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) {
        (void)hipGetLastError();
        return 256;
    }
    cached.store(cus, std::memory_order_relaxed);
    return cus;
}
