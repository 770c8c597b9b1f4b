// Activation checkpoints in 8 bits (ffn.hpp: a signed byte per value and an exponent byte for every 32 columns of a
// row), and GELU's backward pass read from one.
//
// The step of a group is a power of two: x / step and q * step are exact but for the one rounding to an integer, so a
// checkpoint is the same bits whoever makes it, and its values fit one fp16 piece of an operand plane. The rounding is
// off by half a step at most, that is 1/127 of the group's largest magnitude in the worst case (a step just above what
// the magnitude needs) and 1/254 in the best.
//
// Bound by HBM: 5.03 B per value saved or loaded, 9.03 B for the backward pass. Measured at 8192 x 4096: 7.4, 5.8 and 6.2
// TB/s; at 8192 x 4097, where rows start anywhere: 4.1, 5.0 and 5.7.
#include "ffn.hpp"

namespace slb_ffn {

constexpr int kThreads = 256;

// Columns a multiple of 32 and aligned buffers: rows run on without a break in groups, so the tensor is one long row of
// groups. A lane holds four columns, eight lanes a group; a thread has four such quarters of a group in flight, a block's
// threads side by side in each.
constexpr int kAhead = 4;

__global__ void __launch_bounds__(kThreads) k_ck8_save_wide(const float4* __restrict__ x, unsigned* __restrict__ q, unsigned char* __restrict__ eb,
                                                            int64_t quads) {
    const int lane = threadIdx.x & 31;
    const int64_t first = (int64_t)blockIdx.x * (kThreads * kAhead) + threadIdx.x;
    float4 v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; i++)
        if (first + i * kThreads < quads) v[i] = __ldcs(x + first + i * kThreads);
#pragma unroll
    for (int i = 0; i < kAhead; i++) {
        const int64_t at = first + i * kThreads;
        if (at >= quads) break;  // quads is a multiple of eight: the eight lanes of a group leave together
        unsigned top = max(max(__float_as_uint(v[i].x) & 0x7fffffffu, __float_as_uint(v[i].y) & 0x7fffffffu),
                           max(__float_as_uint(v[i].z) & 0x7fffffffu, __float_as_uint(v[i].w) & 0x7fffffffu));
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(0xffu << (lane & 24), top, o));
        const unsigned byte = ck8_exponent(top);
        q[at] = ck8_quantise4(v[i].x, v[i].y, v[i].z, v[i].w, byte);
        if ((lane & 7) == 0) eb[at >> 3] = (unsigned char)byte;
    }
}

template <bool GELU_BWD>
__device__ __forceinline__ Two read_values(const Two& v, const Two& dy) { return GELU_BWD ? mul2(dy, act_grad2(ACT_GELU, v)) : v; }

template <bool GELU_BWD>
__global__ void __launch_bounds__(kThreads) k_ck8_read_wide(const unsigned* __restrict__ q, const unsigned char* __restrict__ eb, const float4* __restrict__ dy,
                                                            float4* __restrict__ out, int64_t quads) {
    const int64_t first = (int64_t)blockIdx.x * (kThreads * kAhead) + threadIdx.x;
    unsigned w[kAhead], byte[kAhead];
    float4 d[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; i++) {
        const int64_t at = first + i * kThreads;
        if (at >= quads) break;
        w[i] = __ldcs(q + at), byte[i] = __ldg(eb + (at >> 3));
        if (GELU_BWD) d[i] = __ldcs(dy + at);
    }
#pragma unroll
    for (int i = 0; i < kAhead; i++) {
        const int64_t at = first + i * kThreads;
        if (at >= quads) break;
        const float step = ck8_step(byte[i]);
        const Two lo = read_values<GELU_BWD>(mul2(Two{ck8_integer<0>(w[i]), ck8_integer<1>(w[i])}, both(step)), GELU_BWD ? Two{d[i].x, d[i].y} : both(0.0f));
        const Two hi = read_values<GELU_BWD>(mul2(Two{ck8_integer<2>(w[i]), ck8_integer<3>(w[i])}, both(step)), GELU_BWD ? Two{d[i].z, d[i].w} : both(0.0f));
        const float4 o = make_float4(lo.x, lo.y, hi.x, hi.y);
        __stcs(out + at, o);
    }
}

// Any columns, any alignment: a warp takes 128 columns of a row, four groups, a lane four of them; kStrips such strips in
// flight. QUADS: rows and buffers allow the four at once. (8192 x 4097: 86 us with a warp per group.)
constexpr int kStrips = 2;
template <bool QUADS, class Index>
__global__ void __launch_bounds__(kThreads) k_ck8_save(const float* __restrict__ x, char* __restrict__ ck, int64_t rows, Index cols) {
    const int lane = threadIdx.x & 31;
    const Index strips = (cols + 127) / 128, first = ((Index)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * kStrips;
    unsigned char* eb = reinterpret_cast<unsigned char*>(ck) + ck8_exp_offset(rows, cols);
    Index row = first / strips, strip = first - row * strips;
    float v[kStrips][4];
    int64_t at[kStrips], group[kStrips];
    int have[kStrips];
#pragma unroll
    for (int i = 0; i < kStrips; i++) {
        const Index col = strip * 128 + lane * 4;
        have[i] = (int64_t)row >= rows || col >= cols ? 0 : cols - col < 4 ? (int)(cols - col) : 4;
        at[i] = (int64_t)row * cols + col, group[i] = (int64_t)row * ck8_groups(cols) + col / kGroup;
        if (QUADS && have[i] == 4) {
            const float4 w = __ldcs(reinterpret_cast<const float4*>(x + at[i]));
            v[i][0] = w.x, v[i][1] = w.y, v[i][2] = w.z, v[i][3] = w.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) v[i][j] = j < have[i] ? __ldg(x + at[i] + j) : 0.0f;
        }
        if (++strip == strips) strip = 0, row++;
    }
#pragma unroll
    for (int i = 0; i < kStrips; i++) {
        unsigned top = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) top = max(top, __float_as_uint(v[i][j]) & 0x7fffffffu);
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const unsigned byte = ck8_exponent(top), q = ck8_quantise4(v[i][0], v[i][1], v[i][2], v[i][3], byte);
        if (QUADS && have[i] == 4) {
            *reinterpret_cast<unsigned*>(ck + at[i]) = q;
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (j < have[i]) ck[at[i] + j] = (char)(q >> (8 * j));
        }
        if ((lane & 7) == 0 && have[i] > 0) eb[group[i]] = (unsigned char)byte;
    }
}

// Aligned buffers, any columns from 32 up: values run on without a break even where groups do not, so a thread takes eight
// neighbours wherever they lie. One division a thread, and one or two groups but where a row ends in a short one.
// (4096 x 2305: 23 us with a lookup for each value of a quad, 33 with a warp per group.)
template <bool GELU_BWD, class Index>
__global__ void __launch_bounds__(kThreads) k_ck8_read_flat(const uint2* __restrict__ q, const unsigned char* __restrict__ eb, const float* __restrict__ dy,
                                                            float* __restrict__ out, Index total, Index cols) {
    const Index groups = (cols + kGroup - 1) / kGroup, at = ((Index)blockIdx.x * kThreads + threadIdx.x) * 8;
    if (at >= total) return;
    const int have = total - at < 8 ? (int)(total - at) : 8;
    const Index row = at / cols, col = at - row * cols;
    const Index group = row * groups + col / kGroup;
    const int in_group = (int)(kGroup - col % kGroup), in_row = cols - col < 8 ? (int)(cols - col) : 8, first = in_group < in_row ? in_group : in_row;
    // values first.. lie in the next group, and, if that one is a row's last and short, from `second` on in the one behind it
    const Index col1 = first == in_row && first < 8 ? 0 : col + first;
    const int second = first + (cols - col1 < 8 ? (int)(cols - col1) : 8);
    const float step0 = ck8_step(__ldg(eb + group)), step1 = first < have ? ck8_step(__ldg(eb + group + 1)) : 0.0f,
                step2 = second < have ? ck8_step(__ldg(eb + group + 2)) : 0.0f;
    uint2 w;
    float d[8];
    if (have == 8) {
        w = __ldcs(q + (at >> 3));
        if (GELU_BWD) {
            const float4 x = __ldcs(reinterpret_cast<const float4*>(dy + at)), y = __ldcs(reinterpret_cast<const float4*>(dy + at) + 1);
            d[0] = x.x, d[1] = x.y, d[2] = x.z, d[3] = x.w, d[4] = y.x, d[5] = y.y, d[6] = y.z, d[7] = y.w;
        }
    } else {
        const unsigned char* bytes = reinterpret_cast<const unsigned char*>(q);
        w = make_uint2(0u, 0u);
        for (int i = 0; i < have; i++) (i < 4 ? w.x : w.y) |= (unsigned)bytes[at + i] << (8 * (i & 3));
        if (GELU_BWD) {
#pragma unroll
            for (int i = 0; i < 8; i++) d[i] = i < have ? dy[at + i] : 0.0f;
        }
    }
    float o[8];
    o[0] = ck8_integer<0>(w.x), o[1] = ck8_integer<1>(w.x), o[2] = ck8_integer<2>(w.x), o[3] = ck8_integer<3>(w.x);
    o[4] = ck8_integer<0>(w.y), o[5] = ck8_integer<1>(w.y), o[6] = ck8_integer<2>(w.y), o[7] = ck8_integer<3>(w.y);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const Two step = Two{i < first ? step0 : i < second ? step1 : step2, i + 1 < first ? step0 : i + 1 < second ? step1 : step2};
        const Two r = read_values<GELU_BWD>(mul2(Two{o[i], o[i + 1]}, step), GELU_BWD ? Two{d[i], d[i + 1]} : both(0.0f));
        o[i] = r.x, o[i + 1] = r.y;
    }
    if (have == 8) {
        __stcs(reinterpret_cast<float4*>(out + at), make_float4(o[0], o[1], o[2], o[3]));
        __stcs(reinterpret_cast<float4*>(out + at) + 1, make_float4(o[4], o[5], o[6], o[7]));
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < have) out[at + i] = o[i];
    }
}

// Any columns, any alignment: a warp per group, a lane per column, four groups of a warp in flight.
constexpr int kAheadAny = 4;
template <bool GELU_BWD>
__global__ void __launch_bounds__(kThreads) k_ck8_read(const char* __restrict__ ck, const float* __restrict__ dy, float* __restrict__ out, int64_t rows,
                                                       int64_t cols) {
    const int lane = threadIdx.x & 31;
    const int64_t groups = ck8_groups(cols), first = ((int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * kAheadAny;
    const unsigned char* eb = reinterpret_cast<const unsigned char*>(ck) + ck8_exp_offset(rows, cols);
    int64_t row = first / groups, g = first - row * groups, at[kAheadAny];
    float d[kAheadAny];
    int q[kAheadAny];
    unsigned byte[kAheadAny];
#pragma unroll
    for (int i = 0; i < kAheadAny; i++) {
        at[i] = row < rows && g * kGroup + lane < cols ? row * cols + g * kGroup + lane : -1;
        if (at[i] >= 0) {
            q[i] = (signed char)__ldg(ck + at[i]);
            byte[i] = __ldg(eb + first + i);
            if (GELU_BWD) d[i] = __ldcs(dy + at[i]);
        }
        if (++g == groups) g = 0, row++;
    }
#pragma unroll
    for (int i = 0; i < kAheadAny; i++)
        if (at[i] >= 0) out[at[i]] = read_values<GELU_BWD>(both((float)q[i] * ck8_step(byte[i])), both(GELU_BWD ? d[i] : 0.0f)).x;
}

static bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
static bool flat(const void* ck, const float* a, const float* b) { return aligned(ck, 8) && aligned(a, 16) && aligned(b, 16); }
static bool wide(int64_t cols, const void* ck, const float* a, const float* b) { return cols % kGroup == 0 && flat(ck, a, b); }
static unsigned wide_grid(int64_t rows, int64_t cols) { return (unsigned)((rows * cols / 4 + kThreads * kAhead - 1) / (kThreads * kAhead)); }
static unsigned any_grid(int64_t rows, int64_t cols) {
    const int64_t per_block = kThreads / 32 * kAheadAny;
    return (unsigned)((rows * ck8_groups(cols) + per_block - 1) / per_block);
}

cudaError_t launch_ck8_save(const float* x, char* ck, int64_t rows, int64_t cols, cudaStream_t st) {
    if (wide(cols, ck, x, nullptr))
        k_ck8_save_wide<<<wide_grid(rows, cols), kThreads, 0, st>>>(reinterpret_cast<const float4*>(x), reinterpret_cast<unsigned*>(ck),
                                                                  reinterpret_cast<unsigned char*>(ck) + ck8_exp_offset(rows, cols), rows * cols / 4);
    else {
        const int64_t warps = (rows * ((cols + 127) / 128) + kStrips - 1) / kStrips;
        const unsigned grid = (unsigned)((warps + kThreads / 32 - 1) / (kThreads / 32));
        const bool quads = cols % 4 == 0 && flat(ck, x, nullptr);
        if (rows * ((cols + 127) / 128) < (int64_t(1) << 30)) {
            if (quads) k_ck8_save<true, unsigned><<<grid, kThreads, 0, st>>>(x, ck, rows, (unsigned)cols);
            else k_ck8_save<false, unsigned><<<grid, kThreads, 0, st>>>(x, ck, rows, (unsigned)cols);
        } else {
            if (quads) k_ck8_save<true, int64_t><<<grid, kThreads, 0, st>>>(x, ck, rows, cols);
            else k_ck8_save<false, int64_t><<<grid, kThreads, 0, st>>>(x, ck, rows, cols);
        }
    }
    return cudaPeekAtLastError();
}
template <bool GELU_BWD>
static cudaError_t launch_read(const char* ck, const float* dy, float* out, int64_t rows, int64_t cols, cudaStream_t st) {
    if (wide(cols, ck, dy, out))
        k_ck8_read_wide<GELU_BWD><<<wide_grid(rows, cols), kThreads, 0, st>>>(reinterpret_cast<const unsigned*>(ck),
                                                                            reinterpret_cast<const unsigned char*>(ck) + ck8_exp_offset(rows, cols),
                                                                            reinterpret_cast<const float4*>(dy), reinterpret_cast<float4*>(out), rows * cols / 4);
    else if (cols >= kGroup && flat(ck, dy, out)) {
        const int64_t total = rows * cols;
        const unsigned grid = (unsigned)(((total + 7) / 8 + kThreads - 1) / kThreads);
        const uint2* q = reinterpret_cast<const uint2*>(ck);
        const unsigned char* eb = reinterpret_cast<const unsigned char*>(ck) + ck8_exp_offset(rows, cols);
        if (total < (int64_t(1) << 31)) k_ck8_read_flat<GELU_BWD, unsigned><<<grid, kThreads, 0, st>>>(q, eb, dy, out, (unsigned)total, (unsigned)cols);
        else k_ck8_read_flat<GELU_BWD, int64_t><<<grid, kThreads, 0, st>>>(q, eb, dy, out, total, cols);
    } else
        k_ck8_read<GELU_BWD><<<any_grid(rows, cols), kThreads, 0, st>>>(ck, dy, out, rows, cols);
    return cudaPeekAtLastError();
}
cudaError_t launch_ck8_load(const char* ck, float* x, int64_t rows, int64_t cols, cudaStream_t st) { return launch_read<false>(ck, nullptr, x, rows, cols, st); }
cudaError_t launch_ck8_gelu_bwd(const char* ck, const float* dy, float* dx, int64_t rows, int64_t cols, cudaStream_t st) {
    return launch_read<true>(ck, dy, dx, rows, cols, st);
}

}  // namespace slb_ffn
