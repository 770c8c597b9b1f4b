// Activation checkpoints in 8 bits (ffn.hpp: a signed byte per value and an exponent byte for every 32 columns of a
// row), and GELU's backward pass read from one.
//
// The step of a group is a power of two: x / step and q * step are exact but for the one rounding to an integer, so a
// checkpoint is the same bits whoever makes it, and its values fit one fp16 piece of an operand plane. The rounding is
// off by half a step at most, that is 1/127 of the group's largest magnitude in the worst case (a step just above what
// the magnitude needs) and 1/254 in the best.
//
// Bound by HBM: 5.03 B per value saved or loaded, 9.03 B for the backward pass.
#include "ffn.hpp"

namespace slb_ffn {

constexpr int kThreads = 256;

// A warp per group of 32 columns, a lane per column.
__global__ void __launch_bounds__(kThreads) k_ck8_save(const float* __restrict__ x, char* __restrict__ ck, int64_t rows, int64_t cols) {
    const int lane = threadIdx.x & 31;
    const int64_t groups = ck8_groups(cols), total = rows * groups, step = (int64_t)gridDim.x * (kThreads / 32);
    unsigned char* eb = reinterpret_cast<unsigned char*>(ck) + ck8_exp_offset(rows, cols);
    for (int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); i < total; i += step) {
        const int64_t row = i / groups, col = (i - row * groups) * kGroup + lane;
        const float v = col < cols ? x[row * cols + col] : 0.0f;
        const unsigned byte = ck8_exponent(__reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu));
        if (col < cols) ck[row * cols + col] = (char)ck8_quantise(v, ck8_inv_step(byte), byte);
        if (lane == 0) eb[i] = (unsigned char)byte;
    }
}

template <bool GELU_BWD>
__global__ void __launch_bounds__(kThreads) k_ck8_read(const char* __restrict__ ck, const float* __restrict__ dy, float* __restrict__ out,
                                                       int64_t rows, int64_t cols) {
    const int lane = threadIdx.x & 31;
    const int64_t groups = ck8_groups(cols), total = rows * groups, step = (int64_t)gridDim.x * (kThreads / 32);
    const unsigned char* eb = reinterpret_cast<const unsigned char*>(ck) + ck8_exp_offset(rows, cols);
    for (int64_t i = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); i < total; i += step) {
        const int64_t row = i / groups, col = (i - row * groups) * kGroup + lane;
        if (col >= cols) continue;
        const float v = (float)(signed char)ck[row * cols + col] * ck8_step(eb[i]);
        out[row * cols + col] = GELU_BWD ? dy[row * cols + col] * act_grad(ACT_GELU, v) : v;
    }
}

static int grid_for(int64_t rows, int64_t cols, int sm_count) {
    const int64_t need = (rows * ck8_groups(cols) + kThreads / 32 - 1) / (kThreads / 32), most = 16 * (int64_t)sm_count;
    return (int)(need < most ? need : most);
}

cudaError_t launch_ck8_save(const float* x, char* ck, int64_t rows, int64_t cols, int sm_count, cudaStream_t st) {
    k_ck8_save<<<grid_for(rows, cols, sm_count), kThreads, 0, st>>>(x, ck, rows, cols);
    return cudaPeekAtLastError();
}
cudaError_t launch_ck8_load(const char* ck, float* x, int64_t rows, int64_t cols, int sm_count, cudaStream_t st) {
    k_ck8_read<false><<<grid_for(rows, cols, sm_count), kThreads, 0, st>>>(ck, nullptr, x, rows, cols);
    return cudaPeekAtLastError();
}
cudaError_t launch_ck8_gelu_bwd(const char* ck, const float* dy, float* dx, int64_t rows, int64_t cols, int sm_count, cudaStream_t st) {
    k_ck8_read<true><<<grid_for(rows, cols, sm_count), kThreads, 0, st>>>(ck, dy, dx, rows, cols);
    return cudaPeekAtLastError();
}

}  // namespace slb_ffn
