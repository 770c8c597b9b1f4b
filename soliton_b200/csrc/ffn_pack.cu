// Operand planes for the products (ffn.hpp): the largest magnitude of each tensor, then fp32 values (or a checkpoint's,
// or the gradient that an activation hands back) as scaled fp16 pieces in the tensor cores' block layout.
//
// The tensor cores have no fp32. A value times a power of two, t = x * 2^(15 - E) with |x| < 2^E,
// is cut into hi = fp16(t) and lo = fp16(t - hi): 22 bits of x wherever |x| > 2^(E - 17), and an absolute error of
// 2^(E - 40) below that. A product of two such values takes three fp16 products, hi*hi + hi*lo + lo*hi; the dropped
// lo*lo is below 2^-22 of it. TF32 pieces would need three products too, at half the rate; bf16 pieces six for the
// the same bits. The price is E, known only after all it covers has been seen. Forward, where both operands' rows are
// rows of the output or its columns, each row has its own and one read is enough. Backward the sums run across rows, so E
// is the tensor's: one more read, which leaves part of it in L2 for the second. A bound serves as well as the maximum
// (17 binades of full precision are far more than needed), so dy * act'(pre) is bounded from dy alone and the gated
// gradients from the three tensors' own maxima.
//
// Large tensors do not stay in L2, and there the second read costs what the first did (38 of 352 us for the gated block's
// gradients at 8192 x 2048 x 768). Their maxima are sampled, a sixteenth of the tensor, and E is taken kMargin higher: a
// value may then exceed the sample's largest by 2^kMargin, and full precision still reaches
// 2^(17 - kMargin) below. The pass that cuts the values keeps their true maximum, and a last pass, which otherwise ends at
// once, does a plane again from the true maximum if it did overflow.
// Infinities and NaN do not count towards a maximum; as operands they become infinities and NaN.
//
// Bound by HBM: 4 B read and 4 B written per value for the plane; backward 4 B more read for the maximum.
#include <cuda_fp16.h>

#include "ffn.hpp"

namespace slb_ffn {

constexpr int kThreads = 256;
// Blocks of k_pack on one SM: two rows of three tensors take 80 registers a thread, of two 64.
template <bool GATED>
constexpr int kPackPerSM = GATED ? 3 : 4;

// ---------------------------------------------------------------- maxima

// Maxima of magnitudes as bit patterns: for finite floats they order as the values do.
__device__ __forceinline__ unsigned finite_bits(float x) {
    const unsigned b = __float_as_uint(x) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}
__device__ __forceinline__ unsigned finite_byte(unsigned byte) { return byte == 255u ? 0u : byte; }

// SAMPLED: some of the tensors are.
template <bool SAMPLED>
__global__ void __launch_bounds__(kThreads) k_amax(const __grid_constant__ AmaxArgs a) {
    stream_next();
    stream_wait();
    const int s = blockIdx.y;
    const AmaxSlot& t = a.slot[s];
    if ((int)blockIdx.x >= t.parts) return;
    unsigned top = 0;
    const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x, step = (int64_t)t.parts * kThreads;
    if (SAMPLED && blockIdx.x == 0 && s == 0 && threadIdx.x < kMaxPlanes) a.tops[threadIdx.x] = 0;
    if (t.is_ck8) {
        const unsigned char* p = static_cast<const unsigned char*>(t.p);
        for (int64_t i = at; i < t.n; i += step) top = max(top, finite_byte(p[i]));
    } else if (SAMPLED && t.sampled) {  // a 16-byte word a thread of 4 KiB in every 64; only where a tensor has many of those
        const float4* w = reinterpret_cast<const float4*>((reinterpret_cast<uintptr_t>(t.p) + 15) & ~(uintptr_t)15);
        const int64_t strips = (t.n - 4) / 16384;
#pragma unroll 4
        for (int64_t i = blockIdx.x; i < strips; i += t.parts) {
            const float4 v = __ldg(w + i * 4096 + threadIdx.x);
            top = max(max(top, max(finite_bits(v.x), finite_bits(v.y))), max(finite_bits(v.z), finite_bits(v.w)));
        }
    } else {
        const float* p = static_cast<const float*>(t.p);
        // up to three values ahead of the first 16-byte boundary, then 128-bit words, then the rest
        int64_t head = (int64_t)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / 4;
        if (head > t.n) head = t.n;
        const int64_t words = (t.n - head) / 4;
        const float4* w = reinterpret_cast<const float4*>(p + head);
        int64_t i = at;
        for (; i + 3 * step < words; i += 4 * step) {
            float4 v[4];
#pragma unroll
            for (int u = 0; u < 4; u++) v[u] = __ldg(w + i + u * step);
#pragma unroll
            for (int u = 0; u < 4; u++)
                top = max(max(top, max(finite_bits(v[u].x), finite_bits(v[u].y))), max(finite_bits(v[u].z), finite_bits(v[u].w)));
        }
        for (; i < words; i += step) {
            const float4 v = __ldg(w + i);
            top = max(max(top, max(finite_bits(v.x), finite_bits(v.y))), max(finite_bits(v.z), finite_bits(v.w)));
        }
        if (at < head) top = max(top, finite_bits(p[at]));
        if (at < t.n - head - 4 * words) top = max(top, finite_bits(p[head + 4 * words + at]));
    }
    __shared__ unsigned part[kThreads / 32];
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
    __syncthreads();
    if (threadIdx.x < 32) {
        top = __reduce_max_sync(0xffffffffu, threadIdx.x < kThreads / 32 ? part[threadIdx.x] : 0u);
        if (threadIdx.x == 0) a.parts[s * kAmaxParts + blockIdx.x] = __uint_as_float(top);
    }
}

// E with every finite |x| < 2^E: from the largest magnitude's bits, or the largest exponent byte (|q| <= 127 < 2^7).
__device__ __forceinline__ int exponent_of(unsigned top, int is_ck8) {
    if (is_ck8) return (int)top - 127 + 7;
    return (int)(top >> 23) - 126;
}
constexpr int kMargin = 6;
constexpr int kLeastExp = -110, kMostExp = 128;  // so that 2^(15 - E) and its reciprocal are normal floats

// ---------------------------------------------------------------- planes

struct Eight {
    float v[8];
};
// Eight values from p on, of which `have` exist; `wide`: 16-byte loads may be used.
__device__ __forceinline__ Eight load8(const float* p, int have, bool wide) {
    Eight r;
    if (wide && have == 8) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(p)), y = __ldg(reinterpret_cast<const float4*>(p) + 1);
        r.v[0] = x.x, r.v[1] = x.y, r.v[2] = x.z, r.v[3] = x.w, r.v[4] = y.x, r.v[5] = y.y, r.v[6] = y.z, r.v[7] = y.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) r.v[i] = i < have ? __ldg(p + i) : 0.0f;
    }
    return r;
}
// The same from a checkpoint, whose eight columns from a multiple of eight lie in one group.
__device__ __forceinline__ Eight load8_ck(const signed char* q, const unsigned char* exp, int have, bool wide) {
    const float step = ck8_step(__ldg(exp));
    Eight r;
    if (wide && have == 8) {
        const uint2 w = __ldg(reinterpret_cast<const uint2*>(q));
        r.v[0] = ck8_integer<0>(w.x) * step, r.v[1] = ck8_integer<1>(w.x) * step, r.v[2] = ck8_integer<2>(w.x) * step, r.v[3] = ck8_integer<3>(w.x) * step;
        r.v[4] = ck8_integer<0>(w.y) * step, r.v[5] = ck8_integer<1>(w.y) * step, r.v[6] = ck8_integer<2>(w.y) * step, r.v[7] = ck8_integer<3>(w.y) * step;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) r.v[i] = i < have ? (float)__ldg(q + i) * step : 0.0f;
    }
    return r;
}

__device__ __forceinline__ void split8(const Eight& x, float scale, uint4& hi, uint4& lo) {
    unsigned h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const Two t = mul2(Two{x.v[2 * i], x.v[2 * i + 1]}, both(scale));
        const __half2 p = __floats2half2_rn(t.x, t.y);
        const float2 f = __half22float2(p);
        const Two d = add2(t, Two{-f.x, -f.y});
        const __half2 r = __floats2half2_rn(d.x, d.y);
        h[i] = *reinterpret_cast<const unsigned*>(&p), l[i] = *reinterpret_cast<const unsigned*>(&r);
    }
    hi = make_uint4(h[0], h[1], h[2], h[3]), lo = make_uint4(l[0], l[1], l[2], l[3]);
}

// Row r, eight columns `chunk` of a block.
__device__ __forceinline__ void store_pieces(char* block, int pieces, int r, int chunk, const Eight& x, float scale) {
    uint4 hi, lo;
    split8(x, scale, hi, lo);
    char* at = block + (r >> 3) * (1024 * pieces) + (r & 7) * 128 + ((chunk ^ (r & 7)) << 4);
    *reinterpret_cast<uint4*>(at) = hi;
    if (pieces == 2) *reinterpret_cast<uint4*>(at + 1024) = lo;
}

// Column sums over a block's 64 rows: a thread holds two rows' eight columns; four rows meet in a warp, then the eight
// warps in order.
__device__ __forceinline__ void block_colsum(const Eight (&x)[2], float (&buf)[8][kBlock], float* out, int64_t col0, int64_t cols) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        t[i] = x[0].v[i] + x[1].v[i];
        t[i] += __shfl_xor_sync(0xffffffffu, t[i], 8);
        t[i] += __shfl_xor_sync(0xffffffffu, t[i], 16);
    }
    __syncthreads();  // whoever read `buf` last is done
    if (lane < 8)
#pragma unroll
        for (int i = 0; i < 8; i++) buf[warp][lane * 8 + i] = t[i];
    __syncthreads();
    if (threadIdx.x < kBlock && col0 + threadIdx.x < cols) {
        float sum = buf[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < 8; w++) sum += buf[w][threadIdx.x];
        out[col0 + threadIdx.x] = sum;
    }
}

// Eight columns from element `off`, group `group` on, of a job's operand in fp32 or (ck not null) of its checkpoint.
__device__ __forceinline__ Eight load8_held(const float* p, const void* ck, const unsigned char* exp, int wide, int64_t off, int64_t group, int have) {
    if (have == 0) return load8(nullptr, 0, false);
    return ck ? load8_ck(static_cast<const signed char*>(ck) + off, exp + group, have, wide) : load8(p + off, have, wide);
}

// One block of 64 x 64: a thread takes eight columns of two rows, all of whose loads are issued before the first is used.
// TOP: the largest finite magnitude is wanted as well. SUM: column sums may be.
template <int KIND, bool TOP, bool SUM>
__device__ __forceinline__ void pack_unit(const PackJob& j, int unit, float scale, float (&s_sum)[8][kBlock], unsigned* top) {
    const int chunk = threadIdx.x & 7, row_in = threadIdx.x >> 3;
    const int u = unit - j.first_unit, rb = u / j.col_blocks, cb = u - rb * j.col_blocks;
    const int64_t col = (int64_t)cb * kBlock + chunk * 8;
    const int have = col >= j.cols ? 0 : j.cols - col < 8 ? (int)(j.cols - col) : 8;
    char* block = j.plane + ((int64_t)rb * j.row_stride + cb) * (int64_t)(j.pieces * kImageBytes);
    Eight x[2], y[2], z[2];
    unsigned most = 0;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int64_t row = (int64_t)rb * kBlock + row_in + 32 * h, off = row * j.cols + col;
        const int64_t group = KIND == PACK_FP32 ? 0 : row * j.groups + col / kGroup;
        const int got = row < j.rows ? have : 0;
        if (KIND == PACK_CK8) x[h] = load8_held(nullptr, j.b8, j.b_exp, j.b_wide, off, group, got);
        else x[h] = load8_held(j.a, nullptr, nullptr, j.a_wide, off, 0, got);
        if (KIND == PACK_ACT || KIND == PACK_GATED) y[h] = load8_held(j.b, j.b8, j.b_exp, j.b_wide, off, group, got);
        if (KIND == PACK_GATED) z[h] = load8_held(j.c, j.c8, j.c_exp, j.c_wide, off, group, got);
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int r = row_in + 32 * h;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const Two d = Two{x[h].v[i], x[h].v[i + 1]}, pre = Two{y[h].v[i], y[h].v[i + 1]};
            if (KIND == PACK_ACT) {
                const Two r = mul2(d, act_grad2(j.act, pre));
                x[h].v[i] = r.x, x[h].v[i + 1] = r.y;
            }
            if (KIND == PACK_GATED) {
                Two value, grad;
                act_and_grad2(j.act, pre, value, grad);
                const Two r = mul2(mul2(d, Two{z[h].v[i], z[h].v[i + 1]}), grad), up = mul2(d, value);
                x[h].v[i] = r.x, x[h].v[i + 1] = r.y;
                y[h].v[i] = up.x, y[h].v[i + 1] = up.y;
            }
        }
        if (TOP && KIND != PACK_CK8) {
#pragma unroll
            for (int i = 0; i < 8; i++) most = max(most, KIND == PACK_GATED ? max(finite_bits(x[h].v[i]), finite_bits(y[h].v[i])) : finite_bits(x[h].v[i]));
        }
        store_pieces(block, KIND == PACK_CK8 ? 1 : 2, r, chunk, x[h], scale);
        if (KIND == PACK_GATED) store_pieces(block + (int64_t)j.second * (int64_t)(2 * kImageBytes), 2, r, chunk, y[h], scale);
    }
    if (TOP && KIND != PACK_CK8) {
        most = __reduce_max_sync(0xffffffffu, most);
        if ((threadIdx.x & 31) == 0 && most > *reinterpret_cast<volatile unsigned*>(top)) atomicMax(top, most);
    }
    if (SUM && KIND != PACK_CK8 && j.colsum) block_colsum(x, s_sum, j.colsum + (int64_t)rb * j.cols, (int64_t)cb * kBlock, j.cols);
    if (SUM && KIND == PACK_GATED && j.colsum2) block_colsum(y, s_sum, j.colsum2 + (int64_t)rb * j.cols, (int64_t)cb * kBlock, j.cols);
}

template <bool TOP, bool SUM, bool GATED>
__device__ __forceinline__ void pack_any(const PackJob& j, int unit, int e, float (&s_sum)[8][kBlock], unsigned* tops) {
    const float scale = exp2f((float)(15 - e));
    unsigned* top = tops + j.plane_id;
    if (j.kind == PACK_FP32) pack_unit<PACK_FP32, TOP, SUM>(j, unit, scale, s_sum, top);
    else if (j.kind == PACK_CK8) pack_unit<PACK_CK8, TOP, SUM>(j, unit, scale, s_sum, top);
    else if (!GATED || j.kind == PACK_ACT) pack_unit<PACK_ACT, TOP, SUM>(j, unit, scale, s_sum, top);
    else pack_unit<PACK_GATED, TOP, SUM>(j, unit, scale, s_sum, top);
}

// Blocks of threads take blocks of 64 x 64 round robin over all jobs. SAMPLED: the maxima are. GATED: a job is.
template <bool SAMPLED, bool GATED>
__global__ void __launch_bounds__(kThreads, kPackPerSM<GATED>) k_pack(const __grid_constant__ PackArgs a) {
    __shared__ int s_exp[kMaxSlots];
    __shared__ float s_sum[8][kBlock];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    stream_next();
    stream_wait();
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < a.n_counters; i += kThreads) a.counters[i] = 0;
    if (warp < a.amax.slots) {
        unsigned top = 0;
        for (int i = lane; i < a.amax.slot[warp].parts; i += 32) top = max(top, __float_as_uint(a.amax.parts[warp * kAmaxParts + i]));
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) s_exp[warp] = exponent_of(top, a.amax.slot[warp].is_ck8);
    }
    __syncthreads();
    int ji = 0;
    for (int unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
        while (ji + 1 < a.jobs && unit >= a.job[ji + 1].first_unit) ji++;
        const PackJob& j = a.job[ji];
        int e;
        if (GATED && j.kind == PACK_GATED) {
            e = s_exp[0] + max(s_exp[1] + (j.act != ACT_NONE), s_exp[2]);  // |act'| < 2, |act(g)| <= |g|
        } else if (j.kind == PACK_ACT) {
            e = s_exp[0] + 1;
        } else {
            e = kLeastExp;
            for (int s = 0; s < a.amax.slots; s++)
                if (j.slots >> s & 1) e = max(e, s_exp[s]);
        }
        if (SAMPLED && j.kind != PACK_CK8) e += kMargin;
        e = min(max(e, kLeastExp), kMostExp);
        if (unit == j.first_unit && threadIdx.x == 0) (SAMPLED ? a.guess : a.exps)[j.plane_id] = e;
        pack_any<SAMPLED, true, GATED>(j, unit, e, s_sum, a.amax.tops);
    }
}

// The planes whose largest value did not fit below 2^e. (A checkpoint's exponents are never sampled, so its plane, which
// keeps no maximum, always fits.)
template <bool GATED>
__global__ void __launch_bounds__(kThreads, kPackPerSM<GATED>) k_repack(const __grid_constant__ PackArgs a) {
    __shared__ float s_sum[8][kBlock];
    stream_next();
    stream_wait();
    int e[kMaxPlanes];
    bool again[kMaxPlanes], any = false;
    for (int p = 0; p < kMaxPlanes; p++) {
        const int got = a.planes >> p & 1 ? a.guess[p] : 0, need = min(max(exponent_of(a.amax.tops[p], 0), kLeastExp), kMostExp);
        again[p] = (a.planes >> p & 1) && need > got;
        e[p] = again[p] ? need : got;
        any |= again[p];
        if (blockIdx.x == 0 && threadIdx.x == 0 && (a.planes >> p & 1)) a.exps[p] = e[p];
    }
    if (!any) return;
    int ji = 0;
    for (int unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
        while (ji + 1 < a.jobs && unit >= a.job[ji + 1].first_unit) ji++;
        const PackJob& j = a.job[ji];
        const int p = j.plane_id;
        if (p == 0 ? again[0] : p == 1 ? again[1] : again[2]) pack_any<false, false, GATED>(j, unit, p == 0 ? e[0] : p == 1 ? e[1] : e[2], s_sum, a.amax.tops);
    }
}
static_assert(kMaxPlanes == 3, "three planes by name above");

// Planes with a scale for each row: WARPS warps take a row and hold it in registers between its maximum and its pieces
// (CHUNKS times 256 values each; with 0, for rows that would not fit, it is read again, from L2). A block takes 8 / WARPS rows.
template <int CHUNKS, int WARPS>
__device__ __forceinline__ void pack_row(const RowJob& j, int64_t row, int part, unsigned* tops) {
    const int lane = threadIdx.x & 31;
    const bool wide = (j.cols & 7) == 0 && (reinterpret_cast<uintptr_t>(j.a) & 15) == 0;
    const int chunks = j.col_blocks * 8, first = part * 32 + lane;
    const float* src = j.a + row * j.cols;
    const bool there = row < j.rows;
    const auto fetch = [&](int c) {
        const int64_t left = there ? j.cols - (int64_t)c * 8 : 0;
        return load8(src + (int64_t)c * 8, left <= 0 ? 0 : left < 8 ? (int)left : 8, wide);
    };
    Eight x[CHUNKS > 0 ? CHUNKS : 1];
    unsigned top = 0;
    if (CHUNKS > 0) {
#pragma unroll
        for (int i = 0; i < CHUNKS; i++) x[i] = fetch(first + 32 * WARPS * i);
#pragma unroll
        for (int i = 0; i < CHUNKS; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) top = max(top, finite_bits(x[i].v[e]));
    } else {
#pragma unroll 4
        for (int c = first; c < chunks; c += 32 * WARPS) {
            const Eight y = fetch(c);
#pragma unroll
            for (int e = 0; e < 8; e++) top = max(top, finite_bits(y.v[e]));
        }
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (WARPS > 1) {
        const int warp = threadIdx.x >> 5;
        if (lane == 0) tops[warp] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WARPS; w++) top = max(top, tops[warp / WARPS * WARPS + w]);
    }
    const int e = min(max(exponent_of(top, 0), kLeastExp), kMostExp);
    const float scale = exp2f((float)(15 - e));
    if (first == 0) j.factor[row] = exp2f((float)(j.is_a ? e - 30 : e));
    char* base = j.plane + (row >> 6) * j.col_blocks * (int64_t)(2 * kImageBytes);
    const auto put = [&](int c, const Eight& y) { store_pieces(base + (int64_t)(c >> 3) * (int64_t)(2 * kImageBytes), 2, (int)(row & 63), c & 7, y, scale); };
    if (CHUNKS > 0) {
#pragma unroll
        for (int i = 0; i < CHUNKS; i++)
            if (first + 32 * WARPS * i < chunks) put(first + 32 * WARPS * i, x[i]);
    } else {
#pragma unroll 4
        for (int c = first; c < chunks; c += 32 * WARPS) put(c, fetch(c));
    }
}
template <int CHUNKS, int WARPS>
__global__ void __launch_bounds__(kThreads) k_rows(const __grid_constant__ RowArgs a) {
    __shared__ unsigned tops[kThreads / 32];
    stream_next();
    stream_wait();
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < a.n_counters; i += kThreads) a.counters[i] = 0;
    const int group = (int)blockIdx.x / WARPS, warp = threadIdx.x >> 5;
    int ji = a.jobs - 1;
    while (group < a.job[ji].first_group) ji--;
    const RowJob& j = a.job[ji];
    pack_row<CHUNKS, WARPS>(j, (int64_t)(group - j.first_group) * 8 + (int)blockIdx.x % WARPS * (8 / WARPS) + warp / WARPS, warp % WARPS, tops);
}
struct RowKernel {
    void (*kernel)(RowArgs);
    int warps;
};
// By the row's blocks of 64 columns, four to a chunk of 256 (8192 x 4096: 64 us read twice by a warp, 38 once by four).
static RowKernel row_kernel(int blocks) {
    if (blocks <= 4) return {k_rows<1, 1>, 1};
    if (blocks <= 8) return {k_rows<2, 1>, 1};
    if (blocks <= 12) return {k_rows<3, 1>, 1};
    if (blocks <= 16) return {k_rows<4, 1>, 1};
    if (blocks <= 32) return {k_rows<4, 2>, 2};
    if (blocks <= 64) return {k_rows<4, 4>, 4};
    if (blocks <= 128) return {k_rows<4, 8>, 8};
    return {k_rows<0, 8>, 8};
}

// A block takes 32 columns, each of its warps every eighth block row; the eight sums meet in order.
__global__ void __launch_bounds__(kThreads) k_colsum(const float* parts, float* out, const float* parts2, float* out2, int count, int64_t cols) {
    __shared__ float part[kThreads / 32][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t j = (int64_t)blockIdx.x * 32 + lane;
    if (blockIdx.y == 1) parts = parts2, out = out2;
    stream_next();
    stream_wait();
    float sum = 0;
    if (j < cols) {
#pragma unroll 8
        for (int i = warp; i < count; i += kThreads / 32) sum += parts[(int64_t)i * cols + j];
    }
    part[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && j < cols) {
        sum = part[0][lane];
#pragma unroll
        for (int w = 1; w < kThreads / 32; w++) sum += part[w][lane];
        out[j] = sum;
    }
}

cudaError_t launch_rows(const RowArgs& a, cudaStream_t st) {
    const RowKernel k = row_kernel(a.job[0].col_blocks);  // all jobs have the same
    return launch_early(k.kernel, dim3((unsigned)(a.groups * k.warps)), kThreads, 0, st, 1, a);
}

cudaError_t launch_amax(const AmaxArgs& a, int, cudaStream_t st) {
    int most = 1;
    for (int s = 0; s < a.slots; s++) most = most > a.slot[s].parts ? most : a.slot[s].parts;
    bool sampled = false;
    for (int s = 0; s < a.slots; s++) sampled |= a.slot[s].sampled != 0;
    return launch_early(sampled ? k_amax<true> : k_amax<false>, dim3((unsigned)most, (unsigned)a.slots), kThreads, 0, st, 1, a);
}

static bool gated(const PackArgs& a) { return a.job[0].kind == PACK_GATED; }  // it comes first
static dim3 pack_grid(const PackArgs& a, int sm_count) {
    const int most = sm_count * (gated(a) ? kPackPerSM<true> : kPackPerSM<false>);  // as many as run at once: each starts with the maxima
    return dim3((unsigned)(a.units < most ? a.units : most));
}
static void set_access(PackArgs& a) {
    const auto aligned = [](const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
    for (int i = 0; i < a.jobs; i++) {
        PackJob& j = a.job[i];
        const bool whole = (j.cols & 7) == 0;
        j.groups = ck8_groups(j.cols);
        j.a_wide = whole && aligned(j.a, 16);
        j.b_wide = whole && (j.b8 ? aligned(j.b8, 8) : aligned(j.b, 16));
        j.c_wide = whole && (j.c8 ? aligned(j.c8, 8) : aligned(j.c, 16));
        j.b_exp = j.b8 ? static_cast<const unsigned char*>(j.b8) + ck8_exp_offset(j.rows, j.cols) : nullptr;
        j.c_exp = j.c8 ? static_cast<const unsigned char*>(j.c8) + ck8_exp_offset(j.rows, j.cols) : nullptr;
    }
}
cudaError_t launch_pack(PackArgs& a, int sm_count, cudaStream_t st) {
    set_access(a);
    const auto kernel = gated(a) ? (a.sampled ? k_pack<true, true> : k_pack<false, true>) : (a.sampled ? k_pack<true, false> : k_pack<false, false>);
    return launch_early(kernel, pack_grid(a, sm_count), kThreads, 0, st, 1, a);
}
cudaError_t launch_repack(const PackArgs& a, int sm_count, cudaStream_t st) {
    return launch_early(gated(a) ? k_repack<true> : k_repack<false>, pack_grid(a, sm_count), kThreads, 0, st, 1, a);
}

cudaError_t launch_colsum(const float* parts, float* out, const float* parts2, float* out2, int count, int64_t cols, cudaStream_t st) {
    const bool first = out != nullptr, both = first && out2;
    return launch_early(k_colsum, dim3((unsigned)((cols + 31) / 32), both ? 2u : 1u), kThreads, 0, st, 1, first ? parts : parts2, first ? out : out2, parts2, out2, count,
                        cols);
}

}  // namespace slb_ffn
