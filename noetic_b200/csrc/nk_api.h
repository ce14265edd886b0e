// nk_api.h -- what the C ABI's argument checks share (head_api.cu, train_api.cu):
// the status of a refused call, sizes, alignment and overlaps, the device of a
// call and the copies of the host-array forms.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>
#include <exception>
#include <initializer_list>
#include <new>
#include <string>
#include <vector>

#include "../../include/noetic/head.h"
#include "nk_kernels.h"

namespace {

struct HeadError {
    nk_status code;
    std::string msg;
};

[[noreturn]] inline void fail(nk_status code, const std::string &msg) { throw HeadError{code, msg}; }
inline void need(bool ok, const char *msg) {
    if (!ok) fail(NK_ERR_INVALID, msg);
}

inline void cuda_check(cudaError_t e, const char *what) {
    if (e != cudaSuccess) {
        cudaGetLastError();
        fail(e == cudaErrorMemoryAllocation ? NK_ERR_OOM : NK_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
    }
}

template <class F>
nk_status guard(const char *name, F &&f) {
    try {
        try {
            f();
            return NK_OK;
        } catch (const HeadError &e) {
            nk::set_last_error(std::string(name) + ": " + e.msg);
            return e.code;
        } catch (const std::bad_alloc &) {
            nk::set_last_error("host allocation failed");
            return NK_ERR_OOM;
        } catch (const std::exception &e) {
            nk::set_last_error(e.what());
            return NK_ERR_INVALID;
        }
    } catch (...) {  // the message itself could not be stored
        return NK_ERR_OOM;
    }
}

constexpr uint64_t MAX_ROWS = 1ull << 26;
constexpr uint64_t MAX_WIDTH = 1ull << 30;
constexpr uint32_t NO_TOKEN = 0xFFFFFFFFu;

inline int elem_size(int dtype) { return dtype == NK_F32 ? 4 : 2; }

inline void check_dtype(int dtype) { need(dtype == NK_F32 || dtype == NK_F16 || dtype == NK_BF16, "unknown dtype"); }

inline void check_matrix(uint64_t rows, uint64_t width, uint64_t stride, const char *what) {
    uint64_t n = 0;
    if (rows > MAX_ROWS || width > MAX_WIDTH) fail(NK_ERR_INVALID, std::string(what) + ": rows are limited to 2^26, the width to 2^30");
    if (stride < width) fail(NK_ERR_INVALID, std::string(what) + ": the row stride is below the width");
    if (!nk::checked_mul(rows, stride, n)) fail(NK_ERR_INVALID, std::string(what) + ": rows * stride is limited to 2^37 elements");
}

inline void check_aligned(const void *p, size_t to, const char *what) {
    if (((uintptr_t)p & (to - 1)) != 0) fail(NK_ERR_INVALID, std::string(what) + " is not aligned to its element");
}
inline void check_f32(std::initializer_list<const void *> ps) {
    for (const void *p : ps) check_aligned(p, 4, "an f32 or u32 array");
}

// Whether two matrices of `rows` rows share an element without being the same
// array at the same stride (columns of one wide array are apart).
inline bool overlap(const void *a, uint64_t as, const void *b, uint64_t bs, uint64_t rows, uint64_t width, int es) {
    const uintptr_t pa = (uintptr_t)a, pb = (uintptr_t)b;
    if (pa == pb && (as == bs || rows == 1)) return false;
    const uintptr_t ea = pa + ((rows - 1) * as + width) * es, eb = pb + ((rows - 1) * bs + width) * es;
    if (ea <= pb || eb <= pa) return false;
    if (as != bs) return true;
    const uint64_t gap = pa < pb ? pb - pa : pa - pb, row = as * es, at = gap % row;
    return at < width * es || at + width * es > row;
}

// An array from its first byte to its last.
struct Span {
    const void *p;
    uint64_t bytes;
};
inline Span matrix_span(const void *p, uint64_t rows, uint64_t width, uint64_t stride, int es) {
    return {p, rows ? ((rows - 1) * stride + width) * es : 0};
}
// No output shares a byte with another one or with an input.  (Matrices among
// each other: `overlap`.)
inline void check_apart(std::initializer_list<Span> outs, std::initializer_list<Span> ins) {
    auto meet = [](const Span &a, const Span &b) {
        return a.p && b.p && a.bytes && b.bytes && (uintptr_t)a.p < (uintptr_t)b.p + b.bytes && (uintptr_t)b.p < (uintptr_t)a.p + a.bytes;
    };
    for (const Span *a = outs.begin(); a != outs.end(); ++a) {
        for (const Span *b = a + 1; b != outs.end(); ++b) need(!meet(*a, *b), "two outputs overlap");
        for (const Span &b : ins) need(!meet(*a, b), "an output overlaps an input");
    }
}

// The device that owns the call's first array, current for the call.  All of its
// arrays that are not null have to be there, or managed.
struct OnDevice {
    int before = -1;
    explicit OnDevice(std::initializer_list<const void *> arrays) {
        int device = -1, now = 0;
        for (const void *p : arrays) {
            if (!p) continue;
            cudaPointerAttributes at{};
            cuda_check(cudaPointerGetAttributes(&at, p), "cudaPointerGetAttributes");
            if (at.type == cudaMemoryTypeManaged) continue;
            need(at.type == cudaMemoryTypeDevice, "the arrays must be in device memory");
            if (device < 0) device = at.device;
            need(device == at.device, "the arrays are on different devices");
        }
        if (device < 0) return;
        cuda_check(cudaGetDevice(&now), "cudaGetDevice");
        if (now != device) {
            cuda_check(cudaSetDevice(device), "cudaSetDevice");
            before = now;
        }
    }
    ~OnDevice() {
        if (before >= 0) cudaSetDevice(before);
    }
};

// Device copies of host arrays for the length of one call.
struct HostCall {
    std::vector<void *> own;
    int before = 0;
    explicit HostCall(int device) {
        cuda_check(cudaGetDevice(&before), "cudaGetDevice");
        cuda_check(cudaSetDevice(device), "cudaSetDevice");
    }
    ~HostCall() {
        for (void *p : own) cudaFree(p);
        cudaSetDevice(before);
    }
    template <class T>
    T *room(size_t bytes, bool wanted = true) {
        if (!wanted) return nullptr;
        void *p = nullptr;
        cuda_check(cudaMalloc(&p, bytes ? bytes : 1), "cudaMalloc");
        try {
            own.push_back(p);
        } catch (...) {
            cudaFree(p);
            throw;
        }
        return (T *)p;
    }
    template <class T>
    T *up(const T *host, size_t bytes) {
        if (!host) return nullptr;
        void *p = room<void>(bytes);
        cuda_check(cudaMemcpy(p, host, bytes, cudaMemcpyHostToDevice), "upload");
        return (T *)p;
    }
    void down(void *host, const void *dev, size_t bytes) {
        if (host) cuda_check(cudaMemcpy(host, dev, bytes, cudaMemcpyDeviceToHost), "download");
    }
};

// The status of a nested device call, its message kept.
inline void nested(nk_status st) {
    if (st != NK_OK) fail(st, nk_last_error());
}

inline void check_ids(const uint32_t *ids, uint64_t n, uint64_t vocab) {
    for (uint64_t i = 0; i < n; ++i) need(ids[i] == NO_TOKEN || ids[i] < vocab, "a token id is out of range");
}

}  // namespace
