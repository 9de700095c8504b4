// Operators on device memory: what the entry points with a `cuda_stream` argument launch, and what the training step launches on
// its own stream.  Nothing here allocates, synchronises or keeps anything between calls: outputs and workspaces are the caller's.
#pragma once
#include "common.hpp"

namespace ullis {
namespace dev {

enum { F32 = ULLIS_CUDA_F32, F16 = ULLIS_CUDA_F16, BF16 = ULLIS_CUDA_BF16 };
inline size_t size_of(int dtype) { return dtype == F32 ? 4 : 2; }

struct Stream {   // where a call's kernels go
    ullis_cuda_runtime* rt;
    cudaStream_t stream;
    uint32_t* status;   // two words for a kernel that gives up waiting

    // A kernel whose first statement is chain_entry() (common.hpp), set up while the one before it runs.
    template <typename... P, typename... A>
    void chain(const char* what, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, A... args) const {
        rt->launch_on(stream, true, kernel, grid, block, smem, P(args)...);
        launched(what);
    }
    void launched(const char* what) const {
        if (stream == rt->stream) { rt->launched(what); return; }   // (timing marks are events on that stream)
        ++rt->launches;
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) fail(ULLIS_CUDA_ERR_CUDA, std::string("launch of ") + what + ": " + cudaGetErrorString(e));
    }
};

// A matrix of rows of `channels` elements, `stride` elements apart.
struct Rows {
    const void* data;
    size_t stride;
};

struct Tape8 {   // a tape of [rows, channels] in a buffer of its own
    uint8_t *codes, *exponents;
    Tape8(DeviceBuffer& buffer, size_t rows, size_t channels) {
        const size_t bytes = (rows * channels + 255) / 256 * 256;
        codes = buffer.as<uint8_t>(bytes + rows * ((channels + 31) / 32));
        exponents = codes + bytes;
    }
};

// One CTA waits on a barrier that nothing arrives on, `polls` times, and says so as the products do.
void wait_selftest(const Stream& s, uint32_t polls);

// ---- the 8-bit tape (tape.cuh); codes [rows, channels] and exponents [rows, ceil(channels / 32)] without gaps
void tape_pack(const Stream& s, int dtype, Rows x, size_t rows, size_t channels, uint8_t* codes, uint8_t* exponents);
void tape_unpack(const Stream& s, int dtype, const uint8_t* codes, const uint8_t* exponents, size_t rows, size_t channels, void* x,
                 size_t x_stride);
constexpr size_t TAPE_NORM_CHANNELS = 8192;   // the widest row that the two kernels below keep in registers
void tape_layer_norm(const Stream& s, int dtype, Rows x, const uint16_t* weight, const uint16_t* bias, size_t rows, size_t channels,
                     void* y, uint8_t* codes, uint8_t* exponents);
size_t tape_layer_norm_backward_workspace(const ullis_cuda_runtime* rt, size_t rows, size_t channels);
void tape_layer_norm_backward(const Stream& s, int dtype, const uint8_t* codes, const uint8_t* exponents, Rows gy, const uint16_t* weight,
                              Rows residual, size_t rows, size_t channels, void* gx, float* g_weight, float* g_bias, void* workspace);

// ---- gradient of a linear's weights from the tape of its input: g [out, in] f32 = gy^T . x^ (gy F16 or BF16)
size_t tape_weight_grad_workspace(const ullis_cuda_runtime* rt, size_t rows, size_t in_features, size_t out_features);
void tape_weight_grad(const Stream& s, int dtype, const uint8_t* codes, const uint8_t* exponents, Rows gy, size_t rows,
                      size_t in_features, size_t out_features, float* g, void* workspace);

// ---- cross-entropy of a head with its gradient
struct HeadGrad {
    int dtype;                 // of the products' operands, hidden and the gradients: F16 or BF16
    bool hidden_f32, out_f32;  // hidden comes in f32 (and is rounded to F16); the gradients leave in f32
    bool fold_scale;           // F16: g_weight is that of the weights with their scale, sum of g * hidden; no g_scale
    Rows hidden;               // [rows, channels]
    const uint32_t* bits;      // packed signs, or null and
    const void* weight;        // dense [vocab, channels] of `dtype`
    const uint16_t* scale;     // FP16 [vocab], with bits
    const uint16_t* bias;      // FP16 [vocab], nullable
    const uint32_t* labels;    // [rows]
    uint32_t ignore_id;
    size_t rows, time, channels, vocab;
    float loss_scale;
    float* row_loss;           // [rows]
    void* g_hidden;            // [rows, channels]
    void* g_weight;            // [vocab, channels]
    float *g_scale, *g_bias;   // [vocab], nullable
};
bool head_copies_weight(const void* dense, size_t channels);   // whether the workspace holds the weights as an operand (null: packed)
size_t head_ce_grad_workspace(const ullis_cuda_runtime* rt, size_t rows, size_t channels, size_t vocab, bool copies_weight);
void head_ce_grad(const Stream& s, const HeadGrad& h, void* workspace);

}  // namespace dev
}  // namespace ullis
