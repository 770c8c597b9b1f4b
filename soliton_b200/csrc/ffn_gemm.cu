// fp32-class matrix products over operand planes (ffn.hpp) on the fifth-generation tensor cores.
//
// D = A * B^T over blocks of 64 along K. Per k-block a stage of shared memory receives the blocks of both operands by
// bulk copies (each block is the 8 KiB image the tensor cores read, so a stage is a handful of contiguous copies and no
// tensor map is needed, whatever the matrix's sizes), and one thread issues the products hi*hi, hi*lo, lo*hi of 128 x BN
// x 16 each into an accumulator in tensor memory. K-major and MN-major operands read the same image through different
// descriptors.
//
// The tensor cores round every accumulation towards zero, so a long sum drifts by about half an ulp per step. Sums are
// therefore cut into segments of 256 along K: the accumulator has two buffers, the warps of the epilogue add a finished
// segment to fp32 registers (to nearest) while the next one runs in the other buffer. The same double buffer lets a
// tile's epilogue run under the next tile's products: blocks are persistent, one per SM.
//
// The epilogue transposes 32 x 32 pieces through shared memory so that a lane holds a column: bias, residual, saved
// pre-activations and the result then move as full 128-byte lines at any alignment, and the 32 lanes of a row are one
// group of a checkpoint.
//
// Every wait is bounded: a block whose wait runs out records ST_TIMEOUT_PRODUCT, waits (bounded) for its copies and
// products in flight, frees its tensor memory and returns.
#include "dp_types.h"
#include "ffn.hpp"

namespace slb_ffn {

constexpr int BM = 128, kBlocksM = BM / kBlock;
constexpr int kEpiWarps = 8;
constexpr int kGemmThreads = 128 + 32 * kEpiWarps;          // a warpgroup that copies and issues, two of the epilogue
// Registers: three warpgroups start with 168 a thread, 504 in all; the first keeps 56 and the other two, which hold
// 128 sums a thread, take 224 each: 504 again.
constexpr int kIssueRegs = 56, kEpiRegs = 224;
constexpr int kRingBytes = 192 * 1024;
constexpr int kStageFloats = 32 * 33;                       // one warp's transposition buffer: 32 x 33 or 16 x 65 floats
constexpr int kSmemBytes = kRingBytes + kEpiWarps * kStageFloats * 4 + 256 + 1024;
constexpr int kSegment = 4;                                 // k-blocks per accumulator segment
constexpr int kMaxStages = 4;
constexpr int kGroupM = 8;                                  // row tiles that blocks walk side by side (reuse in L2)

__device__ __forceinline__ unsigned smem_addr(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(unsigned bar, unsigned count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void mbar_expect(unsigned bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(unsigned bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool mbar_try(unsigned bar, unsigned parity) {
    unsigned done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
__device__ __forceinline__ unsigned long long now_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// Waits for the phase; false when the time ran out or (with `stop`) another warp has given up.
__device__ __forceinline__ bool mbar_wait(unsigned bar, unsigned parity, unsigned long long limit_ns, volatile int* stop) {
    if (mbar_try(bar, parity)) return true;
    const unsigned long long began = now_ns();
    for (;;) {
        for (int i = 0; i < 64; i++)
            if (mbar_try(bar, parity)) return true;
        if ((stop && *stop) || now_ns() - began > limit_ns) return false;
    }
}
__device__ __forceinline__ void bulk_load(unsigned dst, const void* src, unsigned bytes, unsigned bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void mma_f16(unsigned d, uint64_t a, uint64_t b, unsigned idesc, unsigned accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
        "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_commit(unsigned bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_load32(unsigned addr, float (&v)[32]) {
    unsigned r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
        "%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
          "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
          "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}

// Shared-memory descriptors of block images (128-byte swizzle, groups of eight 128-byte rows 1 KiB apart). K-major: a
// row is 64 values along K, a step of 16 is 32 bytes. MN-major: a row is 64 values along M or N, eight rows (eight
// steps along K) per group, the next 64 values one image further, a step of 16 is two groups.
template <bool MN>
__device__ __forceinline__ uint64_t descriptor(unsigned image) {
    return (uint64_t)((image & 0x3ffff) >> 4) | (uint64_t)(MN ? kImageBytes >> 4 : 1) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
template <bool MN>
constexpr unsigned kStepBytes = MN ? 2048 : 32;

// ---------------------------------------------------------------- epilogue

struct Piece {          // rows x 32 columns of the output
    int64_t row0, col;  // this lane's column
    int rows;           // that exist
    bool col_ok;
};

// Keeps one row of pre-activations, a column per lane: in fp32, as a checkpoint (the 32 lanes are one group), or both.
__device__ __forceinline__ void save_row(float v, int64_t row, const Piece& p, const GemmArgs& g, float* full, char* ck, int lane) {
    if (full && p.col_ok) full[row * g.cols + p.col] = v;
    if (ck) {
        const float x = p.col_ok ? v : 0.0f;
        const unsigned byte = ck8_exponent(__reduce_max_sync(0xffffffffu, __float_as_uint(x) & 0x7fffffffu));
        if (p.col_ok) ck[row * g.cols + p.col] = (char)ck8_quantise(x, ck8_inv_step(byte), byte);
        if (lane == 0) ck[ck8_exp_offset(g.rows, g.cols) + row * ck8_groups(g.cols) + p.col / kGroup] = (char)byte;
    }
}

// The rows of a piece out of the transposition buffer (`stride` floats a row; the gated pair 32 columns apart), four at a
// time so that their loads are in flight together. Not unrolled further: the epilogue runs once per tile, and straight
// code of its length spends its time fetching instructions (measured: 150 k cycles a tile against 20 k).
template <int EPI, int ROWS>
__device__ __forceinline__ void finish_rows(const GemmArgs& g, const float* buf, const Piece& p, float s1, float s2, int lane) {
    constexpr int kStride = EPI == EPI_GATED ? 65 : 33;
    const bool second = EPI == EPI_STORE && p.row0 >= g.split;
    float* out = second ? g.out2 : g.out;
    const int64_t first = p.row0 - (second ? g.split : 0);
    const float bias = EPI != EPI_STORE && g.bias && p.col_ok ? __ldg(g.bias + p.col) : 0.0f;
    const float bias2 = EPI == EPI_GATED && g.bias2 && p.col_ok ? __ldg(g.bias2 + p.col) : 0.0f;
#pragma unroll 1
    for (int r0 = 0; r0 < ROWS && r0 < p.rows; r0 += 4) {
        float v[4], w[4], add[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            add[i] = EPI == EPI_LINEAR && g.residual && p.col_ok && r0 + i < p.rows ? g.residual[(first + r0 + i) * g.cols + p.col] : 0.0f;
            v[i] = buf[(r0 + i) * kStride + lane] * s1 * s2 + bias;
            if (EPI == EPI_GATED) w[i] = buf[(r0 + i) * kStride + 32 + lane] * s1 * s2 + bias2;
        }
        if (EPI != EPI_STORE && (g.save || g.save8)) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (r0 + i < p.rows) save_row(v[i], first + r0 + i, p, g, g.save, g.save8, lane);
        }
        if (EPI == EPI_GATED && (g.save2 || g.save8_2)) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (r0 + i < p.rows) save_row(w[i], first + r0 + i, p, g, g.save2, g.save8_2, lane);
        }
        if (EPI != EPI_STORE && g.act != ACT_NONE) {
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = act_of(g.act, v[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (EPI == EPI_GATED) v[i] *= w[i];
            if (EPI == EPI_LINEAR && g.residual) v[i] += add[i];
            if (p.col_ok && r0 + i < p.rows) out[(first + r0 + i) * g.cols + p.col] = v[i];
        }
    }
}

// ---------------------------------------------------------------- the kernel

struct Tile {
    int m, n;
};
__device__ __forceinline__ Tile tile_at(int t, int m_tiles, int n_tiles) {
    const int per_group = kGroupM * n_tiles, group = t / per_group, in_group = t - group * per_group;
    const int first = group * kGroupM, height = min(kGroupM, m_tiles - first);
    return Tile{first + in_group % height, in_group / height};
}

// Warp 0 copies, warp 1 issues the products, warps 4 to 11 read the accumulators: two per 32 rows, each half the columns.
template <int BN, int PB, bool AMN, bool BMN, int EPI>
__global__ void __launch_bounds__(kGemmThreads, 1) k_gemm(const __grid_constant__ GemmArgs g) {
    constexpr int kBlocksN = BN / kBlock, kHalf = BN / 2, kChunks = kHalf / 32;
    constexpr int kABytes = kBlocksM * (int)kImageBytes, kBBytes = kBlocksN * (int)kImageBytes;  // of one piece
    constexpr int kStageBytes = 2 * kABytes + PB * kBBytes;
    constexpr int kStages = kRingBytes / kStageBytes < kMaxStages ? kRingBytes / kStageBytes : kMaxStages;
    static_assert(kStages >= 2, "a stage to copy into while one is read");
    extern __shared__ char raw[];
    char* ring = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    float* turn = reinterpret_cast<float*>(ring + kRingBytes);
    uint64_t* bars = reinterpret_cast<uint64_t*>(turn + kEpiWarps * kStageFloats);
    int* words = reinterpret_cast<int*>(bars + 2 * kMaxStages + 5);
    volatile int* stop = words;
    const unsigned ring_at = smem_addr(ring), bar_at = smem_addr(bars);
    const unsigned full = bar_at, empty = full + 8 * kMaxStages, tfull = empty + 8 * kMaxStages, tempty = tfull + 16, drained = tempty + 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; s++) mbar_init(full + 8 * s, 1), mbar_init(empty + 8 * s, 1);
        for (int b = 0; b < 2; b++) mbar_init(tfull + 8 * b, 1), mbar_init(tempty + 8 * b, kEpiWarps);
        mbar_init(drained, 1);
        *stop = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(words + 1)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = *reinterpret_cast<volatile unsigned*>(words + 1);
    const int tiles = g.m_tiles * g.n_tiles;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
        if (warp == 0 && lane == 0) {
            unsigned it = 0;
            bool ok = true;
            for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
                const Tile at = tile_at(t, g.m_tiles, g.n_tiles);
                const int ma = at.m * kBlocksM, na = min(kBlocksM, g.a.mn_blocks - ma);
                int nb;
                int64_t b_at[kBlocksN];
                if (EPI == EPI_GATED) {  // blocks of the two weights by turns
                    const int first = at.n * (kBlocksN / 2);
                    nb = 2 * min(kBlocksN / 2, g.gate_blocks - first);
                    for (int j = 0; j < kBlocksN; j++) b_at[j] = (int64_t)((j & 1) * g.gate_blocks + first + (j >> 1)) * g.b.mn_stride;
                } else {
                    const int first = at.n * kBlocksN;
                    nb = min(kBlocksN, g.b.mn_blocks - first);
                    for (int j = 0; j < kBlocksN; j++) b_at[j] = (int64_t)(first + j) * g.b.mn_stride;
                }
                const unsigned bytes = (unsigned)(na * 2 + nb * PB) * (unsigned)kImageBytes;
                for (int kb = 0; kb < g.k_blocks; kb++, it++) {
                    const unsigned s = it % kStages, round = it / kStages;
                    if (!mbar_wait(empty + 8 * s, (round & 1) ^ 1, g.timeout_ns, stop)) {
                        ok = false;
                        break;
                    }
                    const unsigned bar = full + 8 * s, at_a = ring_at + s * kStageBytes, at_b = at_a + 2 * kABytes;
                    mbar_expect(bar, bytes);
                    for (int i = 0; i < na; i++) {
                        const char* src = g.a.plane + ((int64_t)(ma + i) * g.a.mn_stride + (int64_t)kb * g.a.k_stride) * (int64_t)(2 * kImageBytes);
                        bulk_load(at_a + i * kImageBytes, src, kImageBytes, bar);
                        bulk_load(at_a + kABytes + i * kImageBytes, src + kImageBytes, kImageBytes, bar);
                    }
#pragma unroll
                    for (int j = 0; j < kBlocksN; j++) {
                        if (j >= nb) break;
                        const char* src = g.b.plane + (b_at[j] + (int64_t)kb * g.b.k_stride) * (int64_t)(PB * kImageBytes);
                        bulk_load(at_b + j * kImageBytes, src, kImageBytes, bar);
                        if (PB == 2) bulk_load(at_b + kBBytes + j * kImageBytes, src + kImageBytes, kImageBytes, bar);
                    }
                }
            }
            if (!ok) {  // nothing may still be on its way into this block's shared memory when it ends
                *stop = 1;
                if (g.status) *reinterpret_cast<volatile int*>(g.status) = slb::ST_TIMEOUT_PRODUCT;
                for (unsigned back = it < (unsigned)kStages ? it : (unsigned)kStages; back > 0; back--) {
                    const unsigned i = it - back;
                    mbar_wait(full + 8 * (i % kStages), (i / kStages) & 1, g.timeout_ns, nullptr);
                }
            }
        }
        if (warp == 1 && lane == 0) {
            unsigned it = 0, seg = 0;
            bool ok = true;
            for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
                const Tile at = tile_at(t, g.m_tiles, g.n_tiles);
                const int nb = EPI == EPI_GATED ? 2 * min(kBlocksN / 2, g.gate_blocks - at.n * (kBlocksN / 2)) : min(kBlocksN, g.b.mn_blocks - at.n * kBlocksN);
                const unsigned idesc = 1u << 4 | (AMN ? 1u << 15 : 0u) | (BMN ? 1u << 16 : 0u) | (unsigned)(nb * kBlock >> 3) << 17 | (unsigned)(BM >> 4) << 24;
                for (int k0 = 0; ok && k0 < g.k_blocks; k0 += kSegment, seg++) {
                    const unsigned buf = seg & 1, d = tmem + buf * BN;
                    if (!mbar_wait(tempty + 8 * buf, ((seg >> 1) & 1) ^ 1, g.timeout_ns, stop)) {
                        ok = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const int k1 = min(k0 + kSegment, g.k_blocks);
                    for (int kb = k0; kb < k1; kb++, it++) {
                        const unsigned s = it % kStages;
                        if (!mbar_wait(full + 8 * s, (it / kStages) & 1, g.timeout_ns, stop)) {
                            ok = false;
                            break;
                        }
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const unsigned at_a = ring_at + s * kStageBytes, at_b = at_a + 2 * kABytes;
#pragma unroll
                        for (int product = 0; product < 1 + PB; product++) {  // hi*hi, lo*hi, hi*lo
                            const uint64_t da = descriptor<AMN>(at_a + (product == 1 ? kABytes : 0));
                            const uint64_t db = descriptor<BMN>(at_b + (product == 2 ? kBBytes : 0));
#pragma unroll
                            for (int step = 0; step < kBlock / 16; step++)
                                mma_f16(d, da + (uint64_t)(step * kStepBytes<AMN> >> 4), db + (uint64_t)(step * kStepBytes<BMN> >> 4), idesc,
                                        !(kb == k0 && product == 0 && step == 0));
                        }
                        mma_commit(empty + 8 * s);
                    }
                    if (ok) mma_commit(tfull + 8 * buf);
                }
            }
            if (!ok) {
                *stop = 1;
                if (g.status) *reinterpret_cast<volatile int*>(g.status) = slb::ST_TIMEOUT_PRODUCT;
                mma_commit(drained);
                mbar_wait(drained, 0, g.timeout_ns, nullptr);
            }
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
        const int q = warp & 3, half = (warp >> 2) - 1;  // a warp reads the 32 rows of tensor memory that its number mod 4 gives
        float* buf = turn + (warp - 4) * kStageFloats;
        const int e = g.exps[g.a.exp_id] + g.exps[g.b.exp_id] - 30;  // undo both planes' scaling, in two steps that cannot overflow early
        const float s1 = exp2f((float)(e / 2)), s2 = exp2f((float)(e - e / 2));
        unsigned seg = 0;
        bool ok = true;
        for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
            const Tile at = tile_at(t, g.m_tiles, g.n_tiles);
            float acc[kChunks][32];
#pragma unroll
            for (int c = 0; c < kChunks; c++)
#pragma unroll
                for (int i = 0; i < 32; i++) acc[c][i] = 0.0f;
            for (int k0 = 0; k0 < g.k_blocks; k0 += kSegment, seg++) {
                const unsigned b = seg & 1;
                ok = __all_sync(0xffffffffu, mbar_wait(tfull + 8 * b, (seg >> 1) & 1, g.timeout_ns, stop));
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                for (int c = 0; c < kChunks; c++) {
                    float v[32];
                    tmem_load32(tmem + ((unsigned)(q * 32) << 16) + b * BN + half * kHalf + c * 32, v);
#pragma unroll
                    for (int i = 0; i < 32; i++) acc[c][i] += v[i];
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(tempty + 8 * b);
            }
            if (!ok) break;
            Piece p;
            p.row0 = (int64_t)at.m * BM + q * 32;
            int64_t left = g.rows - p.row0;
            if (EPI == EPI_STORE && p.row0 >= g.split) left += g.split;
            p.rows = left < 0 ? 0 : left < 32 ? (int)left : 32;
            const int all_rows = p.rows;
            const int64_t row0 = p.row0;
#pragma unroll 1
            for (int c = 0; c < (EPI == EPI_GATED ? kChunks / 2 : kChunks); c++) {
                // gated: a half holds 64 columns of the gate, then the same 64 of the second product
                const int64_t col0 = EPI == EPI_GATED ? (int64_t)at.n * kHalf + half * (kHalf / 2) + c * 32 : (int64_t)at.n * BN + half * kHalf + c * 32;
                if (col0 >= g.cols) break;
                p.col = col0 + lane, p.col_ok = p.col < g.cols;
                if (EPI == EPI_GATED) {
#pragma unroll 1
                    for (int pass = 0; pass < 2; pass++) {  // 16 rows of both at a time fit the buffer
                        __syncwarp();
                        if (lane >> 4 == pass) {
                            float* at_row = buf + (lane & 15) * 65;
#pragma unroll
                            for (int u = 0; u < kChunks / 2; u++)
                                if (c == u)
#pragma unroll
                                    for (int i = 0; i < 32; i++) at_row[i] = acc[u][i], at_row[32 + i] = acc[u + kChunks / 2][i];
                        }
                        __syncwarp();
                        p.row0 = row0 + 16 * pass, p.rows = min(16, all_rows - 16 * pass);
                        finish_rows<EPI, 16>(g, buf, p, s1, s2, lane);
                    }
                } else {
                    __syncwarp();
#pragma unroll
                    for (int u = 0; u < kChunks; u++)
                        if (c == u)
#pragma unroll
                            for (int i = 0; i < 32; i++) buf[lane * 33 + i] = acc[u][i];
                    __syncwarp();
                    finish_rows<EPI, 32>(g, buf, p, s1, s2, lane);
                }
            }
        }
        if (!ok && lane == 0) {
            *stop = 1;
            if (g.status) *reinterpret_cast<volatile int*>(g.status) = slb::ST_TIMEOUT_PRODUCT;
        }
        __syncwarp();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

template <int BN, int PB, bool AMN, bool BMN, int EPI>
static cudaError_t launch_one(const GemmArgs& g, int sm_count, cudaStream_t st) {
    static cudaError_t ready = cudaFuncSetAttribute(k_gemm<BN, PB, AMN, BMN, EPI>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    if (ready != cudaSuccess) return ready;
    const int tiles = g.m_tiles * g.n_tiles;
    k_gemm<BN, PB, AMN, BMN, EPI><<<tiles < sm_count ? tiles : sm_count, kGemmThreads, kSmemBytes, st>>>(g);
    return cudaPeekAtLastError();
}

cudaError_t launch_gemm(const GemmArgs& args, bool a_mn, bool b_mn, int pieces_b, Epilogue epi, int sm_count, cudaStream_t st) {
    GemmArgs g = args;
    constexpr int BN = 256;
    const int64_t width = epi == EPI_GATED ? 2 * (int64_t)g.gate_blocks : g.b.mn_blocks;
    g.m_tiles = (g.a.mn_blocks + kBlocksM - 1) / kBlocksM;
    g.n_tiles = (int)((width + BN / kBlock - 1) / (BN / kBlock));
    if (epi == EPI_LINEAR) return launch_one<BN, 2, false, false, EPI_LINEAR>(g, sm_count, st);
    if (epi == EPI_GATED) return launch_one<BN, 2, false, false, EPI_GATED>(g, sm_count, st);
    if (!a_mn && b_mn) return launch_one<BN, 2, false, true, EPI_STORE>(g, sm_count, st);
    if (a_mn && b_mn && pieces_b == 2) return launch_one<BN, 2, true, true, EPI_STORE>(g, sm_count, st);
    if (a_mn && b_mn && pieces_b == 1) return launch_one<BN, 1, true, true, EPI_STORE>(g, sm_count, st);
    return cudaErrorInvalidValue;
}

}  // namespace slb_ffn
