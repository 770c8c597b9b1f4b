// What the feed-forward operators (ffn_api.cu) hand to their kernels: operand planes (ffn_pack.cu), matrix products
// over them (ffn_gemm.cu) and 8-bit activation checkpoints (ck8_kernels.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace slb_ffn {

enum Act : int { ACT_NONE = 0, ACT_GELU = 1, ACT_SILU = 2 };

// ---------------------------------------------------------------- operand planes
//
// A plane holds a rows x cols matrix as fp16 pieces in blocks of 64 x 64, each the image of its values in shared memory as
// the tensor cores read it: groups of eight rows of 128 bytes, a row's eight 16-byte chunks at positions c ^ (row & 7) (the
// 128-byte swizzle). The same image serves as 64 rows of a K-major operand tile and as 64 columns of an MN-major one, so
// one plane feeds every product its matrix appears in, transposed or not. In a plane of two pieces each group's upper 11
// bits (hi, 1 KiB) are followed by the 11 bits after them (lo, 1 KiB). A block is one contiguous copy of 8 KiB a piece. Rows
// and columns beyond the matrix are zero.
constexpr int kBlock = 64;
constexpr size_t kImageBytes = kBlock * kBlock * 2;
constexpr int kAmaxParts = 296;     // partial maxima per tensor at the most, one per block of the maximum's kernel
constexpr int kMaxSlots = 6;        // tensors whose maxima one call needs
constexpr int kMaxJobs = 4;
constexpr int kMaxPlanes = 3;

// One tensor whose largest finite magnitude is wanted, as an exponent: fp32 values, or the exponent bytes of a checkpoint.
struct AmaxSlot {
    const void* p;
    int64_t n;
    int is_ck8;
    int parts;                      // partial maxima, at most kAmaxParts
    int sampled;                    // only a sixteenth is read: 4 KiB in every 64
};
struct AmaxArgs {
    AmaxSlot slot[kMaxSlots];
    int slots;
    float* parts;                   // kMaxSlots x kAmaxParts
    unsigned* tops;                 // zeroed here, for the planes of a sampled maximum
};

enum PackKind : int {
    PACK_FP32 = 0,      // the matrix itself
    PACK_CK8 = 1,       // a checkpoint: one piece holds its values exactly
    PACK_ACT = 2,       // dy * act'(pre), pre in fp32 or a checkpoint
    PACK_GATED = 3,     // dh * u * act'(g) and, into the second half of the plane, dh * act(g)
};
struct PackJob {
    int kind, act;
    const float* a;                 // the matrix, dy or dh
    const float *b, *c;             // pre, or g and u, in fp32 ...
    const void *b8, *c8;            // ... or as checkpoints; `b8` alone with PACK_CK8
    const unsigned char *b_exp, *c_exp;  // their exponent bytes (set by launch_pack, like the next three)
    int a_wide, b_wide, c_wide;     // eight values of a row at a multiple of eight may be read at once
    int64_t groups;
    int64_t rows, cols;
    int row_blocks, col_blocks;     // of this matrix
    int row_stride;                 // blocks per block row of the plane
    int second;                     // PACK_GATED: blocks from a value's block to its partner's
    int pieces;
    char* plane;                    // the matrix's first block
    float* colsum;                  // null, or row_blocks x cols floats: the column sums of each block row
    float* colsum2;                 // the same for PACK_GATED's second matrix
    int slots;                      // bit s: maximum s bounds this job's values (PACK_FP32, PACK_CK8)
    int plane_id;                   // which exponent of `exps` is this plane's
    int first_unit;                 // blocks of the jobs before this one
};
struct PackArgs {
    PackJob job[kMaxJobs];
    int jobs, units;
    AmaxArgs amax;
    int planes;                     // with sampled maxima: all planes of the call have jobs
    int sampled;
    int* guess;                     // sampled: the exponents of the first pass
    int* exps;                      // out: values of plane i were multiplied by 2^(15 - exps[i])
    int* counters;                  // to be zeroed for the products that follow
    int n_counters;
};
// A forward pass's planes: every row has its own scale, so one read of the tensor is enough.
struct RowJob {
    const float* a;
    int64_t rows, cols;
    int col_blocks;
    char* plane;                    // two pieces
    float* factor;                  // out, whole blocks of rows: what undoes a row's scaling, times 2^-30 with `is_a`
    int is_a;
    int first_group;                // groups of eight rows of the jobs before this one
};
struct RowArgs {
    RowJob job[3];
    int jobs, groups;
    int* counters;
    int n_counters;
};

// ---------------------------------------------------------------- products

// Operand: blocks of a plane addressed by (index along M or N, index along K).
struct Operand {
    const char* plane;
    int64_t mn_stride, k_stride;    // in blocks
    int mn_blocks;                  // blocks along M or N that exist
    int exp_id;                     // EPI_STORE: the plane's exponent
};
enum Epilogue : int { EPI_STORE = 0, EPI_LINEAR = 1, EPI_GATED = 2 };
struct GemmArgs {
    Operand a, b;
    int k_blocks;
    int64_t k_len;                  // terms that exist (for the gated block's two products side by side: blocks' worth)
    int m_tiles, n_tiles;           // set by launch_gemm
    const int* exps;                // EPI_STORE
    const float *row_factor, *col_factor, *col_factor2;  // otherwise: of the rows of A and of B (EPI_GATED: of its two weights)
    int whole, slices;              // set by launch_gemm: tiles done by one team, and into how many slices along K the others are cut
    float* partial;                 // sums of those slices (gemm_plan's partial_bytes), and a counter per warp of their tiles, zeroed
    int* counters;
    int* status;                    // sticky status word (host memory), or null
    unsigned long long timeout_ns;  // bound of every wait
    int64_t rows, cols;             // of the output (EPI_GATED: cols of each of the two)
    int64_t split;                  // EPI_STORE: output rows from here on (a multiple of 64) go to out2, counted from 0
    float *out, *out2;
    int act;
    const float *bias, *bias2, *residual;
    float *save, *save2;            // pre-activations in fp32 ...
    char *save8, *save8_2;          // ... or as checkpoints
    int gate_blocks;                // EPI_GATED: blocks of the gate's weight; the second weight's follow in the plane
    int64_t groups, exp_offset;     // set by launch_gemm: of the checkpoints
    int wide;                       // set by launch_gemm: rows and pointers allow 16-byte accesses (8-byte for checkpoints)
};

// How a product is cut, from its sizes in blocks alone (for 148 SMs), so that a dry run knows the scratch.
struct GemmPlan {
    int ctas;                       // 1: tiles of 128 x 128 by single blocks; 2: 256 x 256 by pairs
    int m_tiles, n_tiles;
    int whole, slices;
    size_t partial_bytes;
    int counters;
};
// store: a plain product (EPI_STORE)
GemmPlan gemm_plan(int64_t m_blocks, int64_t n_blocks, int64_t k_blocks, bool store);
// Whether two plain products are small enough to run in one launch: blocks of one tile or slice each, two an SM at the most.
bool side_by_side(const GemmPlan& dx, const GemmPlan& dw);

cudaError_t launch_rows(const RowArgs& a, cudaStream_t st);
cudaError_t launch_amax(const AmaxArgs& a, int sm_count, cudaStream_t st);
cudaError_t launch_pack(PackArgs& a, int sm_count, cudaStream_t st);
// After a pack with sampled maxima: does planes again whose values went beyond what their exponent allows.
cudaError_t launch_repack(const PackArgs& a, int sm_count, cudaStream_t st);
// out[j] = the sum over `parts` of the block rows' column sums, in order; the same for a second matrix where given
cudaError_t launch_colsum(const float* parts, float* out, const float* parts2, float* out2, int count, int64_t cols, cudaStream_t st);
// dx (A K-major, B MN-major) and dw (both MN-major) in one launch, where side_by_side() says so; they need partial sums and
// counters of their own.
cudaError_t launch_gemm_pair(const GemmArgs& dx, const GemmArgs& dw, int pieces_b, cudaStream_t st, int& launches);
// a_mn, b_mn: the operand's blocks hold K along their rows. pieces_b: 1 when B is a checkpoint's plane.
cudaError_t launch_gemm(const GemmArgs& g, bool a_mn, bool b_mn, int pieces_b, Epilogue epi, int sm_count, cudaStream_t st);

// ---------------------------------------------------------------- checkpoints in 8 bits

constexpr int kGroup = 32;
inline __host__ __device__ int64_t ck8_groups(int64_t cols) { return (cols + kGroup - 1) / kGroup; }
inline __host__ __device__ int64_t ck8_exp_offset(int64_t rows, int64_t cols) { return (rows * cols + 15) / 16 * 16; }
inline __host__ __device__ int64_t ck8_bytes(int64_t rows, int64_t cols) {
    return ck8_exp_offset(rows, cols) + rows * ck8_groups(cols);
}
cudaError_t launch_ck8_save(const float* x, char* ck, int64_t rows, int64_t cols, cudaStream_t st);
cudaError_t launch_ck8_load(const char* ck, float* x, int64_t rows, int64_t cols, cudaStream_t st);
cudaError_t launch_ck8_gelu_bwd(const char* ck, const float* dy, float* dx, int64_t rows, int64_t cols, cudaStream_t st);

#ifdef __CUDACC__
// A launch that may begin while the kernel before it drains; what it does before stream_wait() must not touch memory that
// kernel writes or reads.
template <class... Params, class... Args>
inline cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t st, int cluster, Args&&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid, cfg.blockDim = dim3((unsigned)threads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster, attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<Args&&>(args)...);
}
__device__ __forceinline__ void stream_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void stream_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// The exponent byte of a group whose largest magnitude has these bits (sign cleared): the smallest e >= -126 with
// 127 * 2^e >= the magnitude, plus 127; 255 when the group holds an infinity or a NaN. In a normal magnitude
// 1.f * 2^p, 127 * 2^(p - 6) = 1.984375 * 2^p suffices up to f = 0.984375 and 2^(p - 5) is needed beyond.
__device__ __forceinline__ unsigned ck8_exponent(unsigned bits) {
    const unsigned byte = max((bits + 0x1ffffu) >> 23, 7u) - 6u;  // the addition carries into the exponent for f beyond 0.984375
    return bits >= 0x7f800000u ? 255u : byte;
}
// 2^(byte - 127) for bytes 1..254; a byte of 0 stands for 2^-127; 255 gives NaN.
__device__ __forceinline__ float ck8_step(unsigned byte) {
    return byte == 255u ? __int_as_float(0x7fc00000) : byte == 0u ? __int_as_float(0x00400000) : __int_as_float((int)(byte << 23));
}
// The reciprocal step, a power of two as well: bytes that ck8_exponent gives are 1..249, so 254 - byte is 5..253.
__device__ __forceinline__ float ck8_inv_step(unsigned byte) { return __int_as_float((int)(((254u - byte) & 255u) << 23)); }
// Nearest multiple of the step, ties to even, in the low byte; |x| <= 127 steps by the choice of the exponent. x * inv_step
// is exact, and the sum with 1.5 * 2^23 has the integer, rounded, in its low bits. Groups marked 255 store zeros.
__device__ __forceinline__ unsigned ck8_quantise(float x, unsigned byte) {
    return byte == 255u ? 0u : (unsigned)__float_as_int(fmaf(x, ck8_inv_step(byte), 12582912.0f));
}
__device__ __forceinline__ unsigned ck8_quantise4(float x, float y, float z, float w, unsigned byte) {
    const float inv = ck8_inv_step(byte);
    const unsigned lo = __byte_perm(__float_as_uint(fmaf(x, inv, 12582912.0f)), __float_as_uint(fmaf(y, inv, 12582912.0f)), 0x0040);
    const unsigned hi = __byte_perm(__float_as_uint(fmaf(z, inv, 12582912.0f)), __float_as_uint(fmaf(w, inv, 12582912.0f)), 0x0040);
    return byte == 255u ? 0u : __byte_perm(lo, hi, 0x5410);
}

// The J-th of a word's four values: its byte, moved to 0..255, is the low end of 2^23, whose subtraction is exact. (The
// conversion instruction runs at a quarter of the rate.)
template <int J>
__device__ __forceinline__ float ck8_integer(unsigned word) {
    return __uint_as_float(__byte_perm(word ^ 0x80808080u, 0x4b000000u, 0x7440 + J)) - 8388736.0f;
}

// Two floats an instruction.
struct Two {
    float x, y;
};
#define SLB_TWO(name, op)                                                                                                                            \
    __device__ __forceinline__ Two name(const Two& a, const Two& b) {                                                                                \
        Two r;                                                                                                                                       \
        asm("{\n\t.reg .b64 a, b, r;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t" op " r, a, b;\n\tmov.b64 {%0, %1}, r;\n\t}"                        \
            : "=f"(r.x), "=f"(r.y)                                                                                                                   \
            : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));                                                                                               \
        return r;                                                                                                                                    \
    }
SLB_TWO(mul2, "mul.rn.f32x2")
SLB_TWO(add2, "add.rn.f32x2")
#undef SLB_TWO
__device__ __forceinline__ Two fma2(const Two& a, const Two& b, const Two& c) {
    Two r;
    asm("{\n\t.reg .b64 a, b, c, r;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 r, a, b, c;\n\tmov.b64 {%0, %1}, r;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ Two both(float v) { return Two{v, v}; }
// 2^x and 1 / x to two ulps, subnormal results as zero.
__device__ __forceinline__ Two exp2_2(const Two& v) {
    Two r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(v.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(v.y));
    return r;
}
__device__ __forceinline__ Two rcp2(const Two& v) {
    Two r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(v.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(v.y));
    return r;
}

// What an argument's rounding adds to an exponential is relative to terms that vanish with it.
__device__ __forceinline__ Two sigmoid2(const Two& v) { return rcp2(add2(both(1.0f), exp2_2(mul2(v, both(-1.44269504f))))); }
// Phi(v) and e = exp(-v^2 / 2). 1 - erf(z) = (a1 t + ... + a5 t^5) exp(-z^2) with t = 1 / (1 + p z), for z >= 0 (Abramowitz and
// Stegun 7.1.26), is off by 1.5e-7 at most, which Phi halves: about an ulp of a value near one, at under half the
// instructions of erff, whose cost showed (30 k cycles a tile of 128 x 256 against 24 k), and the derivative needs e anyway.
__device__ __forceinline__ Two normal_cdf2(const Two& v, Two& e) {
    e = exp2_2(mul2(mul2(v, v), both(-0.72134752f)));
    const Two t = rcp2(fma2(Two{fabsf(v.x), fabsf(v.y)}, both(0.23164189f), both(1.0f)));  // p / sqrt(2)
    Two h = fma2(t, both(0.5307027145f), both(-0.7265760135f));                             // half the coefficients
    h = fma2(t, h, both(0.7107068705f)), h = fma2(t, h, both(-0.142248368f)), h = fma2(t, h, both(0.127414796f));
    const Two half = add2(both(0.5f), mul2(mul2(t, h), Two{-e.x, -e.y}));  // 1/2 - Phi(-|v|)
    return add2(both(0.5f), Two{copysignf(half.x, v.x), copysignf(half.y, v.y)});
}
__device__ __forceinline__ Two act2(int act, const Two& v) {
    if (act == ACT_GELU) {
        Two e;
        return mul2(v, normal_cdf2(v, e));
    }
    return act == ACT_SILU ? mul2(v, sigmoid2(v)) : v;
}
__device__ __forceinline__ Two act_grad2(int act, const Two& v) {
    if (act == ACT_GELU) {  // Phi(v) + v phi(v)
        Two e;
        const Two cdf = normal_cdf2(v, e);
        return fma2(mul2(v, both(0.39894228f)), e, cdf);
    }
    if (act == ACT_SILU) {
        const Two sig = sigmoid2(v);
        return mul2(sig, fma2(v, Two{1.0f - sig.x, 1.0f - sig.y}, both(1.0f)));
    }
    return both(1.0f);
}
// SiLU and its derivative share the sigmoid.
__device__ __forceinline__ void act_and_grad2(int act, const Two& v, Two& value, Two& grad) {
    if (act == ACT_GELU) {
        Two e;
        const Two cdf = normal_cdf2(v, e);
        value = mul2(v, cdf), grad = fma2(mul2(v, both(0.39894228f)), e, cdf);
    } else if (act == ACT_SILU) {
        const Two sig = sigmoid2(v);
        value = mul2(v, sig), grad = mul2(sig, fma2(v, Two{1.0f - sig.x, 1.0f - sig.y}, both(1.0f)));
    } else {
        value = v, grad = both(1.0f);
    }
}
#endif

}  // namespace slb_ffn
