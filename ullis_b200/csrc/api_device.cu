// extern "C" entry points of the operators on device memory (include/ullis_cuda.h): checks of the arguments, the caller's stream
// and device.  No C++ exception leaves this file.
#include <cmath>
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

// Bytes of a workspace; the text of a refusal is ullis_cuda_last_error(NULL)'s.
template <typename F>
int32_t workspace_of(const ullis_cuda_runtime* rt, size_t* bytes, F&& body) {
    if (!rt || !bytes) {
        set_global_error(rt ? "bytes is null" : "runtime handle is null");
        return ULLIS_CUDA_ERR_ARG;
    }
    *bytes = 0;
    try {
        *bytes = body();
        return ULLIS_CUDA_OK;
    } catch (const Error& e) {
        set_global_error(e.msg.c_str());
        return e.code;
    } catch (const std::exception& e) {
        set_global_error(e.what());
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
void need_sm100(const ullis_cuda_runtime* rt) {
    if (rt->cc_major != 10) fail(ULLIS_CUDA_ERR_CUDA, "this operator needs the tensor cores of an sm_100 device");
}
void need_codes(const uint8_t* codes, const uint8_t* exponents) {
    need_array(codes, "codes", 1);
    need_array(exponents, "exponents", 1);
}

// The tiles of a product are counted in 32 bits, each with up to 16 ranges of K; more, of 2^14 terms and up to 2^10, only the head takes,
// where K is above 2^18 and the other side of its piece of g below 2^10.
void need_tiles(size_t m, size_t n, const char* what) {
    if ((m + 255) / 256 * ((n + 255) / 256) >= ((size_t)1 << 27)) fail(ULLIS_CUDA_ERR_SHAPE, std::string(what) + " shape overflow");
}
void need_product(size_t rows, size_t in_features, size_t out_features) {
    const char* what = "tape weight gradient";
    need_sizes(rows, in_features, what);
    need_sizes(rows, out_features, what);
    need_tiles(out_features, in_features, what);
}
void need_head(size_t rows, size_t channels, size_t vocab) {
    const char* what = "head cross-entropy";
    need_sizes(rows, channels, what);
    need_sizes(rows, vocab, what);
    // (each 1024 rows of the list of those that count look at all labels before them)
    if (rows > (size_t)1 << 24) fail(ULLIS_CUDA_ERR_SHAPE, std::string(what) + " takes at most 2^24 rows");
    need_tiles(rows, vocab, what);
    need_tiles(rows, channels, what);
    need_tiles(vocab, channels, what);
}

}  // namespace

extern "C" {

int32_t ullis_cuda_runtime_wait_selftest_on(ullis_cuda_runtime* rt, void* cuda_stream, uint32_t polls) {
    return on_stream(rt, cuda_stream, [&](const dev::Stream& s) {
        if (polls == 0 || polls > (1u << 20)) fail(ULLIS_CUDA_ERR_ARG, "polls must be in 1..2^20");
        dev::wait_selftest(s, polls);
    });
}

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
    return workspace_of(rt, bytes, [&] {
        need_norm(rows, channels);
        return dev::tape_layer_norm_backward_workspace(rt, rows, channels);
    });
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

int32_t ullis_cuda_tape_weight_grad_workspace(const ullis_cuda_runtime* rt, size_t rows, size_t in_features, size_t out_features,
                                              size_t* bytes) {
    return workspace_of(rt, bytes, [&] {
        need_product(rows, in_features, out_features);
        return dev::tape_weight_grad_workspace(rt, rows, in_features, out_features);
    });
}

int32_t ullis_cuda_tape_weight_grad(ullis_cuda_runtime* rt, void* cuda_stream, int32_t dtype, const uint8_t* codes,
                                    const uint8_t* exponents, const void* gy, size_t gy_stride, size_t rows, size_t in_features,
                                    size_t out_features, float* g, void* workspace, size_t workspace_bytes) {
    return on_stream(rt, cuda_stream, [&](const dev::Stream& s) {
        need_dtype(dtype, false);
        need_product(rows, in_features, out_features);
        need_stride(gy_stride, out_features, "gy");
        need_array(g, "g", 4);
        if (rows == 0) {
            ULLIS_CUDA_CHECK(cudaMemsetAsync(g, 0, in_features * out_features * 4, s.stream));
            return;
        }
        need_codes(codes, exponents);
        need_array(gy, "gy", 2);
        need_workspace(workspace, workspace_bytes, dev::tape_weight_grad_workspace(rt, rows, in_features, out_features));
        need_sm100(rt);
        dev::tape_weight_grad(s, dtype, codes, exponents, dev::Rows{gy, gy_stride}, rows, in_features, out_features, g, workspace);
    });
}

int32_t ullis_cuda_head_ce_grad_workspace(const ullis_cuda_runtime* rt, size_t rows, size_t channels, size_t vocab,
                                          int32_t copies_weight, size_t* bytes) {
    return workspace_of(rt, bytes, [&] {
        need_head(rows, channels, vocab);
        return dev::head_ce_grad_workspace(rt, rows, channels, vocab, copies_weight != 0);
    });
}

int32_t ullis_cuda_head_ce_grad(ullis_cuda_runtime* rt, void* cuda_stream, int32_t dtype, const void* hidden, size_t hidden_stride,
                                const uint32_t* bits, const void* weight, const uint16_t* scale, const uint16_t* bias,
                                const uint32_t* labels, uint32_t ignore_id, size_t rows, size_t time, size_t channels, size_t vocab,
                                float loss_scale, float* row_loss, void* g_hidden, void* g_weight, float* g_scale, float* g_bias,
                                void* workspace, size_t workspace_bytes) {
    return on_stream(rt, cuda_stream, [&](const dev::Stream& s) {
        need_dtype(dtype, false);
        need_head(rows, channels, vocab);
        if (time == 0 || time >= ((size_t)1 << 31) || rows % time) fail(ULLIS_CUDA_ERR_SHAPE, "rows must be a multiple of time");
        need_stride(hidden_stride, channels, "hidden");
        if (!std::isfinite(loss_scale)) fail(ULLIS_CUDA_ERR_ARG, "loss_scale is not finite");
        if ((bits != nullptr) == (weight != nullptr)) fail(ULLIS_CUDA_ERR_ARG, "a head is either packed (bits) or dense (weight)");
        if ((bits != nullptr) != (scale != nullptr)) fail(ULLIS_CUDA_ERR_ARG, "a packed head has row scales, a dense one none");
        if (g_scale && !scale) fail(ULLIS_CUDA_ERR_ARG, "g_scale without row scales");
        if (bits) {
            need_array(bits, "bits", 4);
            need_array(scale, "scale", 2);
        } else {
            need_array(weight, "weight", 2);
        }
        if (bias) need_array(bias, "bias", 2);
        need_array(g_weight, "g_weight", 2);
        if (g_scale) need_array(g_scale, "g_scale", 4);
        if (g_bias) need_array(g_bias, "g_bias", 4);
        if (rows == 0) {
            ULLIS_CUDA_CHECK(cudaMemsetAsync(g_weight, 0, vocab * channels * 2, s.stream));
            if (g_scale) ULLIS_CUDA_CHECK(cudaMemsetAsync(g_scale, 0, vocab * 4, s.stream));
            if (g_bias) ULLIS_CUDA_CHECK(cudaMemsetAsync(g_bias, 0, vocab * 4, s.stream));
            return;
        }
        need_array(hidden, "hidden", 2);
        need_array(labels, "labels", 4);
        need_array(row_loss, "row_loss", 4);
        need_array(g_hidden, "g_hidden", 2);
        need_workspace(workspace, workspace_bytes, dev::head_ce_grad_workspace(rt, rows, channels, vocab, dev::head_copies_weight(weight, channels)));
        need_sm100(rt);
        dev::HeadGrad h{};
        h.dtype = dtype;
        h.hidden = dev::Rows{hidden, hidden_stride};
        h.bits = bits;
        h.weight = weight;
        h.scale = scale;
        h.bias = bias;
        h.labels = labels;
        h.ignore_id = ignore_id;
        h.rows = rows;
        h.time = time;
        h.channels = channels;
        h.vocab = vocab;
        h.loss_scale = loss_scale;
        h.row_loss = row_loss;
        h.g_hidden = g_hidden;
        h.g_weight = g_weight;
        h.g_scale = g_scale;
        h.g_bias = g_bias;
        dev::head_ce_grad(s, h, workspace);
    });
}

}  // extern "C"
