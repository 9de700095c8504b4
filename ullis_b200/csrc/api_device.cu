// extern "C" entry points of the operators on device memory (include/ullis_cuda.h): checks of the arguments, the caller's stream
// and device.  No C++ exception leaves this file.
#include <exception>
#include <new>

#include "device_ops.hpp"
#include "tape.cuh"

using namespace ullis;

namespace {

// Runs `body(stream)` with the runtime's device current and puts the caller's back.
template <typename F>
int32_t on_stream(ullis_cuda_runtime* rt, void* cuda_stream, F&& body) {
    if (!rt) {
        set_global_error("runtime handle is null");
        return ULLIS_CUDA_ERR_ARG;
    }
    struct Device {
        int previous = -1, wanted;
        explicit Device(int device) : wanted(device) {
            ULLIS_CUDA_CHECK(cudaGetDevice(&previous));
            if (previous != wanted) ULLIS_CUDA_CHECK(cudaSetDevice(wanted));
        }
        ~Device() {
            if (previous >= 0 && previous != wanted) cudaSetDevice(previous);
        }
    };
    try {
        rt->throw_on_async_status();
        const Device device(rt->device);
        body(dev::Stream{rt, static_cast<cudaStream_t>(cuda_stream), rt->async_status});
        return ULLIS_CUDA_OK;
    } catch (const Error& e) {
        rt->last_error = e.msg;
        return e.code;
    } catch (const std::bad_alloc&) {
        rt->last_error = "host allocation failed";
        return ULLIS_CUDA_ERR_NOMEM;
    } catch (const std::exception& e) {
        rt->last_error = e.what();
        return ULLIS_CUDA_ERR_ARG;
    }
}

void need_array(const void* p, const char* name, size_t align) {
    if (!p) fail(ULLIS_CUDA_ERR_ARG, std::string(name) + " is null");
    if (reinterpret_cast<uintptr_t>(p) % align) fail(ULLIS_CUDA_ERR_ARG, std::string(name) + " is not aligned to its elements");
}
void need_dtype(int32_t dtype, bool f32) {
    if (!(dtype == ULLIS_CUDA_F16 || dtype == ULLIS_CUDA_BF16 || (f32 && dtype == ULLIS_CUDA_F32)))
        fail(ULLIS_CUDA_ERR_ARG, f32 ? "dtype must be F32, F16 or BF16" : "dtype must be F16 or BF16");
}
void need_stride(size_t stride, size_t columns, const char* name) {
    if (stride < columns) fail(ULLIS_CUDA_ERR_SHAPE, std::string(name) + " stride is below the row's length");
}
void need_workspace(const void* workspace, size_t bytes, size_t needed) {
    if (!needed) return;
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256) fail(ULLIS_CUDA_ERR_ARG, "workspace is null or not aligned to 256 bytes");
    if (bytes < needed)
        fail(ULLIS_CUDA_ERR_SHAPE, "workspace too small: " + std::to_string(bytes) + " bytes, " + std::to_string(needed) + " needed");
}
// Kernels count rows, columns and chunks in 32 bits, elements in 64.
void need_sizes(size_t rows, size_t columns, const char* what) {
    if (columns == 0) fail(ULLIS_CUDA_ERR_SHAPE, std::string(what) + " dimensions must be non-zero");
    if (rows >= ((size_t)1 << 31) || columns >= ((size_t)1 << 24)) fail(ULLIS_CUDA_ERR_SHAPE, std::string(what) + " shape overflow");
}
void need_norm(size_t rows, size_t channels) {
    need_sizes(rows, channels, "tape LayerNorm");
    if (channels > dev::TAPE_NORM_CHANNELS) fail(ULLIS_CUDA_ERR_SHAPE, "tape LayerNorm takes at most 8192 channels");
}
void need_codes(const uint8_t* codes, const uint8_t* exponents) {
    need_array(codes, "codes", 1);
    need_array(exponents, "exponents", 1);
}

}  // namespace

extern "C" {

int32_t ullis_cuda_tape_pack(ullis_cuda_runtime* rt, void* cuda_stream, int32_t dtype, const void* x, size_t x_stride, size_t rows,
                             size_t channels, uint8_t* codes, uint8_t* exponents) {
    return on_stream(rt, cuda_stream, [&](const dev::Stream& s) {
        need_dtype(dtype, true);
        need_sizes(rows, channels, "tape");
        need_stride(x_stride, channels, "x");
        if (rows == 0) return;
        need_array(x, "x", dev::size_of(dtype));
        need_codes(codes, exponents);
        dev::tape_pack(s, dtype, dev::Rows{x, x_stride}, rows, channels, codes, exponents);
    });
}

int32_t ullis_cuda_tape_unpack(ullis_cuda_runtime* rt, void* cuda_stream, int32_t dtype, const uint8_t* codes,
                               const uint8_t* exponents, size_t rows, size_t channels, void* x, size_t x_stride) {
    return on_stream(rt, cuda_stream, [&](const dev::Stream& s) {
        need_dtype(dtype, true);
        need_sizes(rows, channels, "tape");
        need_stride(x_stride, channels, "x");
        if (rows == 0) return;
        need_array(x, "x", dev::size_of(dtype));
        need_codes(codes, exponents);
        dev::tape_unpack(s, dtype, codes, exponents, rows, channels, x, x_stride);
    });
}

int32_t ullis_cuda_tape_layer_norm(ullis_cuda_runtime* rt, void* cuda_stream, int32_t dtype, const void* x, size_t x_stride,
                                   const uint16_t* weight, const uint16_t* bias, size_t rows, size_t channels, void* y,
                                   uint8_t* codes, uint8_t* exponents) {
    return on_stream(rt, cuda_stream, [&](const dev::Stream& s) {
        need_dtype(dtype, true);
        need_norm(rows, channels);
        need_stride(x_stride, channels, "x");
        if (rows == 0) return;
        need_array(x, "x", dev::size_of(dtype));
        need_array(weight, "weight", 2);
        need_array(bias, "bias", 2);
        need_array(y, "y", dev::size_of(dtype));
        need_codes(codes, exponents);
        dev::tape_layer_norm(s, dtype, dev::Rows{x, x_stride}, weight, bias, rows, channels, y, codes, exponents);
    });
}

int32_t ullis_cuda_tape_layer_norm_backward_workspace(const ullis_cuda_runtime* rt, size_t rows, size_t channels, size_t* bytes) {
    if (!rt || !bytes) {
        set_global_error(rt ? "bytes is null" : "runtime handle is null");
        return ULLIS_CUDA_ERR_ARG;
    }
    *bytes = 0;
    try {
        need_norm(rows, channels);
    } catch (const Error& e) {
        set_global_error(e.msg.c_str());
        return e.code;
    }
    *bytes = dev::tape_layer_norm_backward_workspace(rt, rows, channels);
    return ULLIS_CUDA_OK;
}

int32_t ullis_cuda_tape_layer_norm_backward(ullis_cuda_runtime* rt, void* cuda_stream, int32_t dtype, const uint8_t* codes,
                                            const uint8_t* exponents, const void* gy, size_t gy_stride, const uint16_t* weight,
                                            const void* residual, size_t residual_stride, size_t rows, size_t channels, void* gx,
                                            float* g_weight, float* g_bias, void* workspace, size_t workspace_bytes) {
    return on_stream(rt, cuda_stream, [&](const dev::Stream& s) {
        need_dtype(dtype, true);
        need_norm(rows, channels);
        need_stride(gy_stride, channels, "gy");
        if (residual) need_stride(residual_stride, channels, "residual");
        need_array(g_weight, "g_weight", 4);
        need_array(g_bias, "g_bias", 4);
        if (rows == 0) {
            ULLIS_CUDA_CHECK(cudaMemsetAsync(g_weight, 0, channels * 4, s.stream));
            ULLIS_CUDA_CHECK(cudaMemsetAsync(g_bias, 0, channels * 4, s.stream));
            return;
        }
        need_codes(codes, exponents);
        need_array(gy, "gy", dev::size_of(dtype));
        need_array(weight, "weight", 2);
        if (residual) need_array(residual, "residual", dev::size_of(dtype));
        need_array(gx, "gx", dev::size_of(dtype));
        if (residual == gx && residual_stride != channels) fail(ULLIS_CUDA_ERR_ARG, "gx may be residual only where its rows have no gaps");
        need_workspace(workspace, workspace_bytes, dev::tape_layer_norm_backward_workspace(rt, rows, channels));
        dev::tape_layer_norm_backward(s, dtype, codes, exponents, dev::Rows{gy, gy_stride}, weight, dev::Rows{residual, residual_stride},
                                      rows, channels, gx, g_weight, g_bias, workspace);
    });
}

}  // extern "C"
