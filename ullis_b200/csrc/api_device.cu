// extern "C" entry points of the operators on device memory (include/ullis_cuda.h): checks of the arguments, the caller's stream
// and device.  No C++ exception leaves this file.
#include <algorithm>
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
void need_embed(size_t rows, size_t channels, size_t vocab) {
    const char* what = "embedding";
    need_sizes(rows, channels, what);
    if (vocab == 0) fail(ULLIS_CUDA_ERR_SHAPE, "embedding dimensions must be non-zero");
    if (vocab >= (size_t)1 << 31) fail(ULLIS_CUDA_ERR_SHAPE, "embedding shape overflow");
}
void need_scale(float scale) {
    if (!std::isfinite(scale)) fail(ULLIS_CUDA_ERR_ARG, "scale is not finite");
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

// What both calls of a head ask of their arguments; false: no rows, and the sums over them are written.
bool need_head_grad(const dev::Stream& s, const dev::HeadGrad& h) {
    need_dtype(h.dtype, false);
    need_head(h.rows, h.channels, h.vocab);
    if (h.time == 0 || h.time >= ((size_t)1 << 31) || h.rows % h.time) fail(ULLIS_CUDA_ERR_SHAPE, "rows must be a multiple of time");
    need_stride(h.hidden.stride, h.channels, "hidden");
    if (!std::isfinite(h.loss_scale)) fail(ULLIS_CUDA_ERR_ARG, "loss_scale is not finite");
    if ((h.bits != nullptr) == (h.weight != nullptr)) fail(ULLIS_CUDA_ERR_ARG, "a head is either packed (bits) or dense (weight)");
    if ((h.bits != nullptr) != (h.scale != nullptr)) fail(ULLIS_CUDA_ERR_ARG, "a packed head has row scales, a dense one none");
    if (h.g_scale && !h.scale) fail(ULLIS_CUDA_ERR_ARG, "g_scale without row scales");
    if (h.bits) {
        need_array(h.bits, "bits", 4);
        need_array(h.scale, "scale", 2);
    } else {
        need_array(h.weight, "weight", 2);
    }
    if (h.bias) need_array(h.bias, "bias", 2);
    need_array(h.g_weight, "g_weight", 2);
    if (h.g_scale) need_array(h.g_scale, "g_scale", 4);
    if (h.g_bias) need_array(h.g_bias, "g_bias", 4);
    if (h.rows == 0) {
        ULLIS_CUDA_CHECK(cudaMemsetAsync(h.g_weight, 0, h.vocab * h.channels * 2, s.stream));
        if (h.g_scale) ULLIS_CUDA_CHECK(cudaMemsetAsync(h.g_scale, 0, h.vocab * 4, s.stream));
        if (h.g_bias) ULLIS_CUDA_CHECK(cudaMemsetAsync(h.g_bias, 0, h.vocab * 4, s.stream));
        return false;
    }
    need_array(h.hidden.data, "hidden", 2);
    need_array(h.row_loss, "row_loss", 4);
    need_array(h.g_hidden, "g_hidden", 2);
    return true;
}
void need_distill(size_t top, float alpha, float temperature) {
    if (top == 0 || top > dev::DISTILL_MOST) fail(ULLIS_CUDA_ERR_SHAPE, "head distillation takes 1 to 256 entries of a row");
    if (!(alpha >= 0.0f && alpha <= 1.0f)) fail(ULLIS_CUDA_ERR_ARG, "alpha must be in 0 .. 1");
    if (!(temperature >= 0.0078125f && temperature <= 128.0f)) fail(ULLIS_CUDA_ERR_ARG, "temperature must be in 1/128 .. 128");
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

int32_t ullis_cuda_embed(ullis_cuda_runtime* rt, void* cuda_stream, int32_t table_dtype, const void* table, size_t table_stride,
                         const uint32_t* tokens, uint32_t ignore_id, float scale, size_t rows, size_t channels, size_t vocab, int32_t dtype,
                         void* y) {
    return on_stream(rt, cuda_stream, [&](const dev::Stream& s) {
        need_dtype(table_dtype, true);
        need_dtype(dtype, true);
        need_embed(rows, channels, vocab);
        need_stride(table_stride, channels, "table");
        need_scale(scale);
        if (rows == 0) return;
        need_array(table, "table", dev::size_of(table_dtype));
        need_array(tokens, "tokens", 4);
        need_array(y, "y", dev::size_of(dtype));
        dev::embed(s, table_dtype, dev::Rows{table, table_stride}, tokens, ignore_id, scale, rows, channels, vocab, dtype, y);
    });
}

int32_t ullis_cuda_embed_grad_workspace(const ullis_cuda_runtime* rt, int32_t dtype, size_t rows, size_t channels, size_t vocab, size_t* bytes) {
    return workspace_of(rt, bytes, [&] {
        need_dtype(dtype, true);
        need_embed(rows, channels, vocab);
        return dev::embed_grad_workspace(rt, rows, channels);
    });
}

int32_t ullis_cuda_embed_grad(ullis_cuda_runtime* rt, void* cuda_stream, int32_t dtype, const uint32_t* tokens, uint32_t ignore_id,
                              const void* gy, size_t gy_stride, size_t rows, size_t channels, size_t vocab, float scale, float* g,
                              void* workspace, size_t workspace_bytes) {
    return on_stream(rt, cuda_stream, [&](const dev::Stream& s) {
        need_dtype(dtype, true);
        need_embed(rows, channels, vocab);
        need_stride(gy_stride, channels, "gy");
        need_scale(scale);
        need_array(g, "g", 4);
        if (rows == 0) {
            ULLIS_CUDA_CHECK(cudaMemsetAsync(g, 0, vocab * channels * 4, s.stream));
            return;
        }
        need_array(tokens, "tokens", 4);
        need_array(gy, "gy", dev::size_of(dtype));
        need_workspace(workspace, workspace_bytes, dev::embed_grad_workspace(rt, rows, channels));
        dev::embed_grad(s, dtype, tokens, ignore_id, dev::Rows{gy, gy_stride}, rows, channels, vocab, scale, g, workspace);
    });
}

int32_t ullis_cuda_top_logits(ullis_cuda_runtime* rt, void* cuda_stream, int32_t dtype, const void* logits, size_t logits_stride, size_t rows,
                              size_t vocab, size_t k, int32_t* ids, void* top) {
    return on_stream(rt, cuda_stream, [&](const dev::Stream& s) {
        need_dtype(dtype, true);
        need_sizes(rows, vocab, "top logits");
        if (k == 0 || k > vocab || k > dev::TOP_MOST)
            fail(ULLIS_CUDA_ERR_SHAPE, "top logits: k must be at least 1 and at most " + std::to_string(std::min(vocab, dev::TOP_MOST)));
        need_stride(logits_stride, vocab, "logits");
        if (rows == 0) return;
        need_array(logits, "logits", dev::size_of(dtype));
        need_array(ids, "ids", 4);
        need_array(top, "top", dev::size_of(dtype));
        dev::top_logits(s, dtype, dev::Rows{logits, logits_stride}, rows, vocab, k, ids, top);
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
        const dev::HeadGrad h{dtype, false,     false, false, {hidden, hidden_stride}, bits,     weight,   scale,    bias,    labels, ignore_id,
                              rows,  time,      channels, vocab, loss_scale,           row_loss, g_hidden, g_weight, g_scale, g_bias};
        if (!need_head_grad(s, h)) return;
        need_array(labels, "labels", 4);
        need_workspace(workspace, workspace_bytes, dev::head_ce_grad_workspace(rt, rows, channels, vocab, dev::head_copies_weight(weight, channels)));
        need_sm100(rt);
        dev::head_ce_grad(s, h, workspace);
    });
}

int32_t ullis_cuda_head_distill_grad_workspace(const ullis_cuda_runtime* rt, size_t rows, size_t channels, size_t vocab, size_t top,
                                               int32_t has_labels, int32_t copies_weight, size_t* bytes) {
    return workspace_of(rt, bytes, [&] {
        need_head(rows, channels, vocab);
        need_distill(top, 1.0f, 1.0f);
        return dev::head_distill_grad_workspace(rt, rows, channels, vocab, top, has_labels != 0, copies_weight != 0);
    });
}

int32_t ullis_cuda_head_distill_grad(ullis_cuda_runtime* rt, void* cuda_stream, int32_t dtype, const void* hidden, size_t hidden_stride,
                                     const uint32_t* bits, const void* weight, const uint16_t* scale, const uint16_t* bias,
                                     const int32_t* top_ids, int32_t top_dtype, const void* top_logits, size_t top, float alpha,
                                     float temperature, const uint32_t* labels, uint32_t ignore_id, size_t rows, size_t time,
                                     size_t channels, size_t vocab, float loss_scale, float* row_loss, void* g_hidden, void* g_weight,
                                     float* g_scale, float* g_bias, void* workspace, size_t workspace_bytes) {
    return on_stream(rt, cuda_stream, [&](const dev::Stream& s) {
        const dev::HeadGrad h{dtype, false,     false, false, {hidden, hidden_stride}, bits,     weight,   scale,    bias,    labels, ignore_id,
                              rows,  time,      channels, vocab, loss_scale,           row_loss, g_hidden, g_weight, g_scale, g_bias};
        need_dtype(top_dtype, true);
        need_distill(top, alpha, temperature);
        if (!need_head_grad(s, h)) return;
        if (labels) need_array(labels, "labels", 4);
        need_array(top_ids, "top_ids", 4);
        need_array(top_logits, "top_logits", dev::size_of(top_dtype));
        need_workspace(workspace, workspace_bytes,
                       dev::head_distill_grad_workspace(rt, rows, channels, vocab, top, labels != nullptr, dev::head_copies_weight(weight, channels)));
        need_sm100(rt);
        dev::head_distill_grad(s, h, dev::Distill{top_ids, top_logits, top_dtype, top, alpha, temperature}, workspace);
    });
}

}  // extern "C"
