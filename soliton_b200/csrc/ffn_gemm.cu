// fp32-class matrix products over operand planes (ffn.hpp) on the fifth-generation tensor cores.
//
// D = A * B^T over blocks of 64 along K. Per k-block a stage of shared memory receives the blocks of both operands by
// bulk copies (each block is the image the tensor cores read, so a stage is a handful of contiguous copies and no tensor map
// is needed, whatever the matrix's sizes), and one thread issues the products lo*hi, hi*hi, hi*lo, 16 terms each, into an
// accumulator in tensor memory. K-major and MN-major operands read the same image through different descriptors.
//
// The tensor cores round every accumulation towards zero, so a long sum drifts, by 0.14 ulps a step on the average. That
// much is given back (segment_gain), and sums are cut into segments of 256 to 384 terms: the accumulator has two buffers, the
// warps of the epilogue add a finished segment to fp32 registers (to nearest) while the next one runs in the other
// buffer. The same double buffer lets a tile's epilogue run under the next tile's products: blocks are persistent, one per
// SM. At 4096 x 4096 x 4096 a tile takes 106 to 120 k cycles, its products alone 98 k.
//
// The epilogue works on the accumulator's own arrangement, a row per lane and 32 columns at a time (one group of a
// checkpoint), and turns pieces of 32 x 32 through shared memory to store them in whole lines.
//
// Forward, the rows of both operands have their own scales, which the epilogue undoes; backward the whole planes'.
//
// Every wait is bounded: a block whose wait runs out records ST_TIMEOUT_PRODUCT, waits (bounded) for its copies and
// products in flight, frees its tensor memory and returns.
#include "dp_types.h"
#include "ffn.hpp"

namespace slb_ffn {

constexpr int BM = 128;
constexpr int kEpiWarps = 8;
constexpr int kGemmThreads = 128 + 32 * kEpiWarps;          // a warpgroup that copies and issues, two of the epilogue
// Registers: three warpgroups start with 168 a thread, 504 in all; the first keeps 40 and the other two, which hold 128
// sums a thread, take 232 each: 504 again. (Four warpgroups of 64 sums each were no faster and left no room for the epilogue.)
constexpr int kIssueRegs = 40, kEpiRegs = 232;
constexpr int kRingBytes = 192 * 1024;
constexpr int kTurnFloats = 32 * 32;                        // one warp's turning buffer
constexpr int kSmemBytes = kRingBytes + kEpiWarps * kTurnFloats * 4 + 256 + 1024;
// k-blocks per accumulator segment, and in a tile's first two: the products can run that far ahead of the previous tile's
// epilogue. At 4096 x 4096 x 1024 with GELU: 4 and 4 take 134 us, 6 and 6 112, 8 and 8 109 for a third more error.
constexpr int kSegment = 4, kFirstSegments = 6;
constexpr int kMaxStages = 4;
constexpr unsigned long long kDrainNs = 2000000000ull;      // bound of the waits for a block's own copies and products at its end
constexpr int kPlanSMs = 148;                               // how products are cut must not depend on the device
constexpr int kGroupM = 8;                                  // row tiles that blocks walk side by side (reuse in L2)

__device__ __forceinline__ unsigned smem_addr(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(unsigned bar, unsigned count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void mbar_expect(unsigned bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(unsigned bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
// CLUSTER: what the other block of a pair wrote before its arrival is to be seen.
template <bool CLUSTER>
__device__ __forceinline__ bool mbar_try(unsigned bar, unsigned parity) {
    unsigned done;
    if (CLUSTER)
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(done)
                     : "r"(bar), "r"(parity)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(done)
                     : "r"(bar), "r"(parity)
                     : "memory");
    return done != 0;
}
// The same shared-memory address in block `rank` of the cluster, and an arrival there.
__device__ __forceinline__ unsigned remote(unsigned addr, unsigned rank) {
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void mbar_arrive_remote(unsigned bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// The same without making this thread's earlier writes to global memory visible first: for what is ordered otherwise.
__device__ __forceinline__ void mbar_arrive_remote_relaxed(unsigned bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ unsigned long long now_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// Waits for the phase; false when the time ran out or (with `stop`) another warp has given up.
template <bool CLUSTER = false>
__device__ __forceinline__ bool mbar_wait(unsigned bar, unsigned parity, unsigned long long limit_ns, volatile int* stop) {
    if (mbar_try<CLUSTER>(bar, parity)) return true;
    const unsigned long long began = now_ns();
    for (;;) {
        for (int i = 0; i < 64; i++)
            if (mbar_try<CLUSTER>(bar, parity)) return true;
        if ((stop && *stop) || now_ns() - began > limit_ns) return false;
    }
}
__device__ __forceinline__ void bulk_load(unsigned dst, const void* src, unsigned bytes, unsigned bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
template <int CTAS>
__device__ __forceinline__ void mma_f16(unsigned d, uint64_t a, uint64_t b, unsigned idesc, unsigned accumulate) {
    if (CTAS == 1)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
                     "r"(idesc), "r"(accumulate)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
                     "r"(idesc), "r"(accumulate)
                     : "memory");
}
// Arrives at `bar` (in both blocks of a pair) once the products issued so far are done.
template <int CTAS>
__device__ __forceinline__ void mma_commit(unsigned bar) {
    if (CTAS == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((unsigned short)3)
                     : "memory");
}
template <int CTAS>
__device__ __forceinline__ void tmem_alloc(unsigned where) {
    if (CTAS == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(where) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(where) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int CTAS>
__device__ __forceinline__ void tmem_free(unsigned addr) {
    if (CTAS == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(addr) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(addr) : "memory");
}
template <int CTAS>
__device__ __forceinline__ void team_sync() {
    if (CTAS == 1) __syncthreads();
    else asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void give_up(const GemmArgs& g, volatile int* stop) {
    *stop = 1;
    if (g.status) *reinterpret_cast<volatile int*>(g.status) = slb::ST_TIMEOUT_PRODUCT;
}
// Adds 16 columns of the warp's 32 rows of tensor memory, times `gain`, to `sum`.
__device__ __forceinline__ void tmem_add16(unsigned addr, float gain, float* sum) {
    unsigned r[16];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        const Two t = fma2(Two{__uint_as_float(r[i]), __uint_as_float(r[i + 1])}, both(gain), Two{sum[i], sum[i + 1]});
        sum[i] = t.x, sum[i + 1] = t.y;
    }
}

// Shared-memory descriptors of blocks (128-byte swizzle; groups of eight 128-byte rows lie 1 KiB apart for each piece).
// K-major: a row is 64 values along K, a step of 16 is 32 bytes. MN-major: a row is 64 values along M or N, eight rows
// (eight steps along K) per group, the next 64 values one block further, a step of 16 is two groups.
template <bool MN, int PIECES>
__device__ __forceinline__ uint64_t descriptor(unsigned block) {
    constexpr unsigned kGroupBytes = 1024 * PIECES, kBlockBytes = (unsigned)kImageBytes * PIECES;
    return (uint64_t)((block & 0x3ffff) >> 4) | (uint64_t)(MN ? kBlockBytes >> 4 : 1) << 16 | (uint64_t)(kGroupBytes >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
template <bool MN, int PIECES>
constexpr unsigned kStepBytes = MN ? 2048 * PIECES : 32;
constexpr unsigned kLoBytes = 1024;  // from a group's hi to its lo

// Blocks of B along N in a column of tiles: all, or at its end as many as exist -- an even number, so that a pair can halve
// it (what is not there is never stored).
template <int CTAS, int EPI>
__device__ __forceinline__ int blocks_wide(const GemmArgs& g, int n) {
    const int most = 2 * CTAS;
    const int left = EPI == EPI_GATED ? 2 * (g.gate_blocks - n * (most / 2)) : g.b.mn_blocks - n * most;
    return left >= most ? most : (left + 1) & ~1;
}
// Where chunk c (32 columns) of a warp's half lies in a tile's accumulator. Gated: by turns columns of the gate and the
// same columns of the second product, which lie 64 further.
template <int EPI, int CHUNKS>
__device__ __forceinline__ constexpr unsigned column_of(int half, int c) {
    if (EPI != EPI_GATED) return (unsigned)(half * CHUNKS + c) * 32;
    const int j = half * (CHUNKS / 2) + c / 2;
    return (unsigned)((j >> 1) * 128 + (j & 1) * 32 + (c & 1) * 64);
}

// ---------------------------------------------------------------- epilogue

// What a segment of `terms` along K lost on the average to rounding towards zero, given back. An accumulation loses half
// an ulp of the sum so far, 0.36 * 2^-23 of it over all mantissas, and the sum so far is half the final one on the
// average: 0.18 * 2^-23 of the segment a step. Measured, 1024 x 1024 results over 768 to 4096 terms, least squares against
// 64 bits: 0.14 for normal factors, 0.15 with a mean of half their deviation, 0.30 where all products are positive, 0.07
// where 95 % of one factor are zeros. With 0.14 the error at 1024 normal terms halves, 1.31e-6 to 0.7e-6 (fp32 sums: 0.57e-6);
// sums that would have been exact come out that much too large instead of those too small.
template <int PB>
__device__ __forceinline__ float segment_gain(int64_t terms) {
    return 1.0f + 0.14f * 1.1920929e-7f * (float)((1 + PB) * (int)((terms + 15) >> 4));
}

struct Piece {          // rows x 32 columns of the output
    int64_t row0, col0;
    int rows;           // that exist
};

__device__ __forceinline__ unsigned magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The accumulator comes a row per lane, and that is how values are scaled, activated and put into checkpoints (32 columns
// of a row are one group). To be stored they are turned: the warp's buffer is 4 KiB, 32 rows of 32 in 16-byte chunks
// whose place within a row is exclusive-ored with the row's low bits, so that neither writing rows nor reading them
// meets bank conflicts. Stored row per lane, a tensor took 8 k cycles a tile for its 32 lines an instruction. Under the
// products, which read shared memory all the time, a load from it takes some 360 cycles: all of a piece are issued at once.
__device__ __forceinline__ int turned(int row, int chunk) { return (row * 8 + (chunk ^ (row & 7))) * 4; }
__device__ __forceinline__ void put_rows(const float (&v)[32], float* buf, int lane) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; i++) *reinterpret_cast<float4*>(buf + turned(lane, i)) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    __syncwarp();
}
// Stores a piece, plus `add` where given: eight lanes a row, four rows an instruction. at: the element of row 0, column 0.
__device__ __forceinline__ void store_wide(const float (&v)[32], float* out, const float* add, int64_t at, int64_t cols, int rows, float* buf, int lane) {
    const int64_t mine = at + (lane >> 3) * cols + (lane & 7) * 4;
    const int left = rows - (lane >> 3);
    float4 x[8];
    if (add) {
        float4 r[8];
#pragma unroll
        for (int i = 0; i < 8; i++) r[i] = 4 * i < left ? *reinterpret_cast<const float4*>(add + mine + 4 * i * cols) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        put_rows(v, buf, lane);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = *reinterpret_cast<const float4*>(buf + turned(4 * i + (lane >> 3), lane & 7));
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = make_float4(x[i].x + r[i].x, x[i].y + r[i].y, x[i].z + r[i].z, x[i].w + r[i].w);
    } else {
        put_rows(v, buf, lane);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = *reinterpret_cast<const float4*>(buf + turned(4 * i + (lane >> 3), lane & 7));
    }
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (4 * i < left) *reinterpret_cast<float4*>(out + mine + 4 * i * cols) = x[i];
}
__device__ __forceinline__ void keep_wide(const float (&v)[32], const Piece& p, int64_t at, const GemmArgs& g, float* full, char* ck, float* buf, int lane) {
    if (full) store_wide(v, full, nullptr, at, g.cols, p.rows, buf, lane);
    if (ck && lane < p.rows) {
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < 32; i++) top = max(top, magnitude(v[i]));
        const unsigned byte = ck8_exponent(top);
        char* q = ck + at + lane * g.cols;
#pragma unroll
        for (int i = 0; i < 32; i += 8)
            *reinterpret_cast<uint2*>(q + i) =
                make_uint2(ck8_quantise4(v[i], v[i + 1], v[i + 2], v[i + 3], byte), ck8_quantise4(v[i + 4], v[i + 5], v[i + 6], v[i + 7], byte));
        ck[g.exp_offset + (p.row0 + lane) * g.groups + p.col0 / kGroup] = (char)byte;
    }
}
// Undoes the operands' scaling, which cannot overflow before the result does: the row's factor is 2^-30 of its magnitude.
// `col` and `bias`: of the 32 columns.
__device__ __forceinline__ void scale_row(float (&v)[32], float row, const float* col, const float* bias) {
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
        const float4 c = *reinterpret_cast<const float4*>(col + i);
        const float4 b = bias ? __ldg(reinterpret_cast<const float4*>(bias + i)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const Two x = fma2(mul2(Two{v[i], v[i + 1]}, both(row)), Two{c.x, c.y}, Two{b.x, b.y});
        const Two y = fma2(mul2(Two{v[i + 2], v[i + 3]}, both(row)), Two{c.z, c.w}, Two{b.z, b.w});
        v[i] = x.x, v[i + 1] = x.y, v[i + 2] = y.x, v[i + 3] = y.y;
    }
}
template <int ACT>
__device__ __forceinline__ void act_row(float (&v)[32]) {
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const Two r = act2(ACT, Two{v[i + j], v[i + j + 1]});
            v[i + j] = r.x, v[i + j + 1] = r.y;
        }
        // eight at a time: all 32 side by side would not fit the registers
        asm volatile("" : "+f"(v[i]), "+f"(v[i + 1]), "+f"(v[i + 2]), "+f"(v[i + 3]), "+f"(v[i + 4]), "+f"(v[i + 5]), "+f"(v[i + 6]), "+f"(v[i + 7]));
        if (i < 24)
            asm volatile("" : "+f"(v[i + 8]), "+f"(v[i + 9]), "+f"(v[i + 10]), "+f"(v[i + 11]), "+f"(v[i + 12]), "+f"(v[i + 13]), "+f"(v[i + 14]), "+f"(v[i + 15]));
    }
}
__device__ __forceinline__ void act_row(int act, float (&v)[32]) {
    if (act == ACT_GELU) act_row<ACT_GELU>(v);
    else if (act == ACT_SILU) act_row<ACT_SILU>(v);
}
// v: columns p.col0 to p.col0 + 31 of row p.row0 + lane (all 32 exist), w: the same of the gated block's second product.
template <int EPI>
__device__ __forceinline__ void finish_wide(const GemmArgs& g, float (&v)[32], float (&w)[32], const Piece& p, float s1, float s2, float* buf, int lane) {
    const bool second = EPI == EPI_STORE && p.row0 >= g.split;
    const int64_t at = (p.row0 - (second ? g.split : 0)) * g.cols + p.col0;
    if (EPI == EPI_STORE) {
#pragma unroll
        for (int i = 0; i < 32; i++) v[i] = v[i] * s1 * s2;
    } else {
        scale_row(v, s1, g.col_factor + p.col0, g.bias ? g.bias + p.col0 : nullptr);
        keep_wide(v, p, at, g, g.save, g.save8, buf, lane);
        act_row(g.act, v);
        if (EPI == EPI_GATED) {
            scale_row(w, s1, g.col_factor2 + p.col0, g.bias2 ? g.bias2 + p.col0 : nullptr);
            keep_wide(w, p, at, g, g.save2, g.save8_2, buf, lane);
#pragma unroll
            for (int i = 0; i < 32; i++) v[i] *= w[i];
        }
    }
    store_wide(v, second ? g.out2 : g.out, EPI == EPI_LINEAR ? g.residual : nullptr, at, g.cols, p.rows, buf, lane);
}

// Any width, any alignment: turned so that a lane holds a column and a row leaves as one run of up to 128 bytes.
__device__ __forceinline__ void turn(float (&v)[32], float* buf, int lane) {
    put_rows(v, buf, lane);
#pragma unroll
    for (int r = 0; r < 32; r++) v[r] = buf[turned(r, lane >> 2) + (lane & 3)];
}
// v[r]: this lane's column of row r
__device__ __forceinline__ void keep_column(const float (&v)[32], int rows, bool ok, int64_t at, int64_t group, const GemmArgs& g, float* full, char* ck, int lane) {
    if (full) {
#pragma unroll
        for (int r = 0; r < 32; r++)
            if (ok && r < rows) full[at + r * g.cols] = v[r];
    }
    if (ck) {
#pragma unroll
        for (int r = 0; r < 32; r++) {
            if (r >= rows) continue;  // the same for the whole warp
            const unsigned byte = ck8_exponent(__reduce_max_sync(0xffffffffu, ok ? magnitude(v[r]) : 0u));
            if (ok) ck[at + r * g.cols] = (char)ck8_quantise(v[r], byte);
            if (lane == 0) ck[g.exp_offset + group + r * g.groups] = (char)byte;
        }
    }
}
template <int EPI>
__device__ __forceinline__ void finish_any(const GemmArgs& g, float (&v)[32], float (&w)[32], const Piece& p, float s1, float s2, float* buf, int lane) {
    const bool second = EPI == EPI_STORE && p.row0 >= g.split;
    const int64_t row = p.row0 - (second ? g.split : 0), col = p.col0 + lane, at = row * g.cols + col;
    const bool ok = col < g.cols;
    float* out = (second ? g.out2 : g.out) + at;
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] *= s1;
    turn(v, buf, lane);
    const float bias = EPI != EPI_STORE && g.bias && ok ? __ldg(g.bias + col) : 0.0f, by = EPI == EPI_STORE ? s2 : g.col_factor[col];
#pragma unroll
    for (int r = 0; r < 32; r++) v[r] = fmaf(v[r], by, bias);
    if (EPI != EPI_STORE) {
        const int64_t group = row * g.groups + p.col0 / kGroup;
        keep_column(v, p.rows, ok, at, group, g, g.save, g.save8, lane);
        act_row(g.act, v);
        if (EPI == EPI_GATED) {
#pragma unroll
            for (int i = 0; i < 32; i++) w[i] *= s1;
            turn(w, buf, lane);
            const float bias2 = g.bias2 && ok ? __ldg(g.bias2 + col) : 0.0f, by2 = g.col_factor2[col];
#pragma unroll
            for (int r = 0; r < 32; r++) w[r] = fmaf(w[r], by2, bias2);
            keep_column(w, p.rows, ok, at, group, g, g.save2, g.save8_2, lane);
#pragma unroll
            for (int r = 0; r < 32; r++) v[r] *= w[r];
        }
        if (EPI == EPI_LINEAR && g.residual) {
            const float* res = g.residual + at;
#pragma unroll
            for (int r0 = 0; r0 < 32; r0 += 16) {
                float add[16];
#pragma unroll
                for (int i = 0; i < 16; i++) add[i] = ok && r0 + i < p.rows ? res[(r0 + i) * g.cols] : 0.0f;
#pragma unroll
                for (int i = 0; i < 16; i++) v[r0 + i] += add[i];
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 32; r++)
        if (ok && r < p.rows) out[r * g.cols] = v[r];
}

// ---------------------------------------------------------------- the kernel

__device__ __forceinline__ int segment_end(int k0, int k_blocks) {
    if (k_blocks <= 2 * kFirstSegments) return k0 == 0 ? (k_blocks + 1) / 2 : k_blocks;
    return min(k0 + (k0 < 2 * kFirstSegments ? kFirstSegments : kSegment), k_blocks);
}

// What a team takes up at a time: a tile, or a slice of one along K. Tiles that would leave most teams idle in the last
// round are cut so that every team has a part -- and come first, so that what joining them costs runs under the products of
// whole tiles.
struct Unit {
    int m, n, k0, k1, slice;        // slice: of all, -1 for a whole tile
};
__device__ __forceinline__ int units_of(const GemmArgs& g) { return g.whole + (g.m_tiles * g.n_tiles - g.whole) * g.slices; }
__device__ __forceinline__ Unit unit_at(int u, const GemmArgs& g) {
    Unit r;
    const int cut = (g.m_tiles * g.n_tiles - g.whole) * g.slices;
    int t = u - cut;
    r.slice = -1, r.k0 = 0, r.k1 = g.k_blocks;
    if (u < cut) {
        r.slice = u;
        const int s = r.slice % g.slices;
        t = g.whole + r.slice / g.slices;
        r.k0 = (int)((int64_t)g.k_blocks * s / g.slices), r.k1 = (int)((int64_t)g.k_blocks * (s + 1) / g.slices);
    }
    const int per_group = kGroupM * g.n_tiles, group = t / per_group, in_group = t - group * per_group;
    const int first = group * kGroupM, height = min(kGroupM, g.m_tiles - first);
    r.m = first + in_group % height, r.n = in_group / height;
    return r;
}

// Where a warp's sums over a slice lie in memory: 32 rows of CHUNKS x 32 columns, four columns of a lane's row together.
// `who` of `warps`: the part of the tile.
template <int CHUNKS>
__device__ __forceinline__ float4* slice_place(float* partial, int slice, int warps, int who, int lane) {
    return reinterpret_cast<float4*>(partial) + ((int64_t)slice * warps + who) * (CHUNKS * 256) + lane;
}
template <int CHUNKS>
__device__ __forceinline__ void put_slice(const GemmArgs& g, const float (&acc)[CHUNKS][32], int slice, int warps, int who, int lane) {
    float4* to = slice_place<CHUNKS>(g.partial, slice, warps, who, lane);
#pragma unroll
    for (int c = 0; c < CHUNKS; c++)
#pragma unroll
        for (int i = 0; i < 8; i++) __stcg(to + (c * 8 + i) * 32, make_float4(acc[c][4 * i], acc[c][4 * i + 1], acc[c][4 * i + 2], acc[c][4 * i + 3]));
}
// The sums go to memory; the warp that comes last adds up all slices, in their order, and has the tile (true). Nobody waits.
template <int CHUNKS>
__device__ __forceinline__ bool add_slices(const GemmArgs& g, float (&acc)[CHUNKS][32], int slice, int warps, int who, int lane) {
    put_slice(g, acc, slice, warps, who, lane);
    __threadfence();
    __syncwarp();
    int before = 0;
    if (lane == 0) before = atomicAdd(g.counters + (slice / g.slices) * warps + who, 1);
    before = __shfl_sync(0xffffffffu, before, 0);
    if (before != g.slices - 1) return false;
    __threadfence();
    const int first = slice - slice % g.slices;
#pragma unroll
    for (int c = 0; c < CHUNKS; c++)
#pragma unroll
        for (int i = 0; i < 32; i++) acc[c][i] = 0.0f;
#pragma unroll 1
    for (int s = 0; s < g.slices; s++) {
        const float4* from = slice_place<CHUNKS>(g.partial, first + s, warps, who, lane);
#pragma unroll
        for (int c = 0; c < CHUNKS; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float4 v = __ldcg(from + (c * 8 + i) * 32);
                acc[c][4 * i] += v.x, acc[c][4 * i + 1] += v.y, acc[c][4 * i + 2] += v.z, acc[c][4 * i + 3] += v.w;
            }
    }
    return true;
}
// With many slices the warps that come last sit on few SMs and have much to read (30 k of 69 k cycles at eight slices of
// 768 x 768 over 8192 terms); plain products leave it to a kernel of its own then.
constexpr int kManySlices = 5;
__device__ __host__ constexpr bool later(int epi, int slices) { return epi == EPI_STORE && slices >= kManySlices; }

// Undoes both planes' scaling, in two steps that cannot overflow before the result does.
__device__ __forceinline__ void plane_scales(const GemmArgs& g, float& s1, float& s2) {
    const int e = g.exps[g.a.exp_id] + g.exps[g.b.exp_id] - 30;
    s1 = exp2f((float)(e / 2)), s2 = exp2f((float)(e - e / 2));
}
// The 32 rows of tile row m, block `rank` of the team, that quadrant q covers, and how many of them exist.
template <int CTAS, int EPI>
__device__ __forceinline__ Piece rows_of(const GemmArgs& g, int m, int rank, int q) {
    Piece p;
    p.row0 = (int64_t)(m * CTAS + rank) * BM + q * 32;
    int64_t left = g.rows - p.row0;
    if (EPI == EPI_STORE && p.row0 >= g.split) left += g.split;
    p.rows = left < 0 ? 0 : left < 32 ? (int)left : 32;
    return p;
}

// The slices' sums, a warp per 32 rows of eight results, a row per lane: grid over tiles, then parts of a tile, then eights.
// (A warp per 32 x 32 left most SMs without work: 14 us for sixteen slices of 32 tiles.)
constexpr int kSliceThreads = 128;
template <int CTAS>
__global__ void __launch_bounds__(kSliceThreads) k_slices(const __grid_constant__ GemmArgs g) {
    constexpr int kEights = 8 * CTAS, kWarps = CTAS * kEpiWarps;
    const int lane = threadIdx.x & 31;
    stream_next();
    stream_wait();
    const int unit = (int)blockIdx.x * (kSliceThreads / 32) + (threadIdx.x >> 5), e = unit % kEights, who = unit / kEights % kWarps, tile = unit / (kEights * kWarps);
    const Unit at = unit_at(tile * g.slices, g);
    const Piece p = rows_of<CTAS, EPI_STORE>(g, at.m, who / kEpiWarps, who & 3);
    const int64_t col = (int64_t)at.n * 128 * CTAS + (who / 4 % 2) * 64 * CTAS + e * 8;
    if (lane >= p.rows || col >= g.cols) return;
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    const float4* from = slice_place<2 * CTAS>(g.partial, tile * g.slices, kWarps, who, lane) + e * 64;
#pragma unroll 8
    for (int s = 0; s < g.slices; s++, from += kWarps * (2 * CTAS * 256)) {
        const float4 x = __ldcg(from), y = __ldcg(from + 32);
        v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w, v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
    }
    float s1, s2;
    plane_scales(g, s1, s2);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = v[i] * s1 * s2;
    const bool second = p.row0 >= g.split;
    float* out = (second ? g.out2 : g.out) + (p.row0 + lane - (second ? g.split : 0)) * g.cols + col;
    if (g.wide && col + 8 <= g.cols) {
        *reinterpret_cast<float4*>(out) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(out + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (col + i < g.cols) out[i] = v[i];
    }
}

// CTAS = 1: a block per tile of 128 x 128. CTAS = 2: a pair of blocks (a cluster) per tile of 256 x 256: each holds 128 rows of A
// and 128 columns' worth of B in its shared memory and 128 rows of the accumulator, and the first issues products that
// read both. Per value fetched a pair computes twice as much, which is what bounds large products: fetching from L2.
// Warp 0 copies, warp 1 issues the products (in a pair's second block: reports arrived stages to the first), warps 4 to
// 11 read the accumulators: two per 32 rows, half the columns each.
// `block` of `blocks`: of those that work on this product.
template <int CTAS, int PB, bool AMN, bool BMN, int EPI>
__device__ __forceinline__ void multiply(const GemmArgs& g, int block, int blocks) {
    constexpr int BN = 128 * CTAS, kBlocksN = BN / kBlock, kChunks = BN / 64;  // chunks of 32 columns a warp
    constexpr unsigned kABlock = 2 * (unsigned)kImageBytes, kBBlock = PB * (unsigned)kImageBytes;
    constexpr int kStageBytes = 2 * (kABlock + kBBlock);  // this block's 128 rows of A and its share of B
    constexpr int kStages = kRingBytes / kStageBytes < kMaxStages ? kRingBytes / kStageBytes : kMaxStages;
    extern __shared__ char raw[];
    char* ring = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    float* turn = reinterpret_cast<float*>(ring + kRingBytes);
    uint64_t* bars = reinterpret_cast<uint64_t*>(turn + kEpiWarps * kTurnFloats);
    int* words = reinterpret_cast<int*>(bars + 3 * kMaxStages + 5);
    volatile int* stop = words;
    const unsigned ring_at = smem_addr(ring), bar_at = smem_addr(bars);
    const unsigned full = bar_at, empty = full + 8 * kMaxStages, peer_full = empty + 8 * kMaxStages, tfull = peer_full + 8 * kMaxStages, tempty = tfull + 16,
                   drained = tempty + 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = CTAS == 2 ? block & 1 : 0;
    const int team = block / CTAS, teams = blocks / CTAS;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; s++) mbar_init(full + 8 * s, 1), mbar_init(empty + 8 * s, 1), mbar_init(peer_full + 8 * s, 1);
        for (int b = 0; b < 2; b++) mbar_init(tfull + 8 * b, 1), mbar_init(tempty + 8 * b, CTAS * kEpiWarps);
        mbar_init(drained, 1);
        *stop = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) tmem_alloc<CTAS>(smem_addr(words + 1));
    stream_wait();  // and no stream_next(): blocks of a following product, each an SM's worth, made this one slower (231 us against 223)
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    team_sync<CTAS>();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = *reinterpret_cast<volatile unsigned*>(words + 1);
    const int units = units_of(g);

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
        if (warp == 0 && lane == 0) {
            unsigned it = 0;
            bool ok = true;
            for (int t = team; ok && t < units; t += teams) {
                const Unit at = unit_at(t, g);
                const int ma = (at.m * CTAS + rank) * 2, na = max(0, min(2, g.a.mn_blocks - ma));
                const int width = blocks_wide<CTAS, EPI>(g, at.n), share = width / CTAS;  // blocks of B: the tile's and this block's
                int64_t b_at[2];
                int nb = 0;
                for (int j = 0; j < share; j++) {
                    const int i = rank * share + j;
                    if (EPI == EPI_GATED) {  // blocks of the two weights by turns
                        b_at[j] = (int64_t)((i & 1) * g.gate_blocks + at.n * (kBlocksN / 2) + (i >> 1)) * g.b.mn_stride;
                        nb = j + 1;
                    } else {
                        b_at[j] = (int64_t)(at.n * kBlocksN + i) * g.b.mn_stride;
                        if (at.n * kBlocksN + i < g.b.mn_blocks) nb = j + 1;
                    }
                }
                const unsigned bytes = (unsigned)na * kABlock + (unsigned)nb * kBBlock;
                for (int kb = at.k0; kb < at.k1; kb++, it++) {
                    const unsigned s = it % kStages, round = it / kStages;
                    if (!mbar_wait(empty + 8 * s, (round & 1) ^ 1, g.timeout_ns, stop)) {
                        ok = false;
                        break;
                    }
                    const unsigned bar = full + 8 * s, at_a = ring_at + s * kStageBytes, at_b = at_a + 2 * kABlock;
                    mbar_expect(bar, bytes);
#pragma unroll
                    for (int i = 0; i < 2; i++)
                        if (i < na)
                            bulk_load(at_a + i * kABlock, g.a.plane + ((int64_t)(ma + i) * g.a.mn_stride + (int64_t)kb * g.a.k_stride) * (int64_t)kABlock, kABlock, bar);
#pragma unroll
                    for (int j = 0; j < 2; j++)
                        if (j < nb) bulk_load(at_b + j * kBBlock, g.b.plane + (b_at[j] + (int64_t)kb * g.b.k_stride) * (int64_t)kBBlock, kBBlock, bar);
                }
            }
            if (!ok) give_up(g, stop);
            // Nothing may still be on its way into this block's shared memory when it ends, whoever else has given up.
            for (unsigned back = it < (unsigned)kStages ? it : (unsigned)kStages; back > 0; back--) {
                const unsigned i = it - back;
                mbar_wait(full + 8 * (i % kStages), (i / kStages) & 1, kDrainNs, nullptr);
            }
        }
        if (warp == 1 && lane == 0 && rank == 0) {
            unsigned it = 0, seg = 0;
            bool ok = true;
            for (int t = team; ok && t < units; t += teams) {
                const Unit at = unit_at(t, g);
                const unsigned idesc = 1u << 4 | (AMN ? 1u << 15 : 0u) | (BMN ? 1u << 16 : 0u) | (unsigned)(blocks_wide<CTAS, EPI>(g, at.n) * kBlock >> 3) << 17 |
                                       (unsigned)(BM * CTAS >> 4) << 24;
                const int k_blocks = at.k1 - at.k0;
                for (int k0 = 0, k1; ok && k0 < k_blocks; k0 = k1, seg++) {
                    k1 = segment_end(k0, k_blocks);
                    const unsigned buf = seg & 1, d = tmem + buf * BN;
                    if (!mbar_wait<CTAS == 2>(tempty + 8 * buf, ((seg >> 1) & 1) ^ 1, g.timeout_ns, stop)) {
                        ok = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    for (int kb = k0; kb < k1; kb++, it++) {
                        const unsigned s = it % kStages;
                        if (!mbar_wait(full + 8 * s, (it / kStages) & 1, g.timeout_ns, stop) ||
                            (CTAS == 2 && !mbar_wait<true>(peer_full + 8 * s, (it / kStages) & 1, g.timeout_ns, stop))) {
                            ok = false;
                            break;
                        }
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const unsigned at_a = ring_at + s * kStageBytes, at_b = at_a + 2 * kABlock;
                        const uint64_t a_hi = descriptor<AMN, 2>(at_a), b_hi = descriptor<BMN, PB>(at_b);
#pragma unroll
                        for (int step = 0; step < kBlock / 16; step++) {
                            const uint64_t da = a_hi + (step * kStepBytes<AMN, 2> >> 4), db = b_hi + (step * kStepBytes<BMN, PB> >> 4);
                            mma_f16<CTAS>(d, da + (kLoBytes >> 4), db, idesc, !(kb == k0 && step == 0));
                            mma_f16<CTAS>(d, da, db, idesc, 1);
                            if (PB == 2) mma_f16<CTAS>(d, da, db + (kLoBytes >> 4), idesc, 1);
                        }
                        mma_commit<CTAS>(empty + 8 * s);
                    }
                    if (ok) mma_commit<CTAS>(tfull + 8 * buf);
                }
            }
            if (!ok) give_up(g, stop);
            mma_commit<CTAS>(drained);  // nor may products still be reading it, or writing tensor memory
            mbar_wait(drained, 0, kDrainNs, nullptr);
        }
        if (CTAS == 2 && warp == 1 && lane == 0 && rank == 1) {
            const unsigned there = remote(peer_full, 0);
            int rounds = 0;
            for (int t = team; t < units; t += teams) {
                const Unit at = unit_at(t, g);
                rounds += at.k1 - at.k0;
            }
            for (int it = 0; it < rounds; it++) {
                const unsigned s = (unsigned)it % kStages;
                if (!mbar_wait(full + 8 * s, ((unsigned)it / kStages) & 1, g.timeout_ns, stop)) {
                    give_up(g, stop);
                    break;
                }
                mbar_arrive_remote(there + 8 * s);
            }
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
        const int q = warp & 3, half = (warp >> 2) - 1;  // a warp reads the 32 rows of tensor memory that its number mod 4 gives
        float* buf = turn + (warp - 4) * kTurnFloats;
        float s1 = 0.0f, s2 = 0.0f;
        if (EPI == EPI_STORE) plane_scales(g, s1, s2);
        unsigned seg = 0;
        bool ok = true;
        for (int t = team; ok && t < units; t += teams) {
            const Unit at = unit_at(t, g);
            float acc[kChunks][32];
#pragma unroll
            for (int c = 0; c < kChunks; c++)
#pragma unroll
                for (int i = 0; i < 32; i++) acc[c][i] = 0.0f;
            if (EPI == EPI_LINEAR && g.residual) {  // into L2 while the products run: a lane a row, this warp's columns
                const int64_t row = (int64_t)(at.m * CTAS + rank) * BM + q * 32 + lane, col = (int64_t)at.n * BN + half * kChunks * 32;
                if (row < g.rows)
                    for (int64_t c = col; c < min(col + kChunks * 32, g.cols); c += 32)
                        asm volatile("prefetch.global.L2 [%0];" ::"l"(g.residual + row * g.cols + c));
            }
            const int k_blocks = at.k1 - at.k0;
            for (int k0 = 0; k0 < k_blocks; k0 = segment_end(k0, k_blocks), seg++) {
                const unsigned b = seg & 1;
                const int64_t from_k = (int64_t)(at.k0 + k0) * kBlock, to_k = (int64_t)(at.k0 + segment_end(k0, k_blocks)) * kBlock;
                const float gain = segment_gain<PB>(min(to_k, g.k_len) - from_k);
                ok = __all_sync(0xffffffffu, mbar_wait(tfull + 8 * b, (seg >> 1) & 1, g.timeout_ns, stop));
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                for (int c = 0; c < kChunks; c++) {
                    const unsigned from = tmem + ((unsigned)(q * 32) << 16) + b * BN + column_of<EPI, kChunks>(half, c);
                    tmem_add16(from, gain, acc[c]), tmem_add16(from + 16, gain, acc[c] + 16);
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    if (CTAS == 1) mbar_arrive(tempty + 8 * b);
                    else mbar_arrive_remote_relaxed(remote(tempty + 8 * b, 0));  // only reads of tensor memory go before it, and those are complete
                }
            }
            if (!ok) break;
            Piece p = rows_of<CTAS, EPI>(g, at.m, rank, q);
            if (p.rows == 0) continue;
            if (at.slice >= 0) {
                const int who = rank * kEpiWarps + warp - 4;
                if (later(EPI, g.slices)) {
                    put_slice(g, acc, at.slice, CTAS * kEpiWarps, who, lane);
                    continue;
                }
                if (!add_slices(g, acc, at.slice, CTAS * kEpiWarps, who, lane)) continue;
            }
            if (EPI != EPI_STORE) s1 = g.row_factor[p.row0 + lane];  // whole blocks of factors exist
            // In place and in a loop that moves the next chunk up: registers are short, and so should the code be, which runs
            // once per tile and is bound by fetching it when it is long (150 k cycles a tile for four chunks in a row).
            constexpr int kTaken = EPI == EPI_GATED ? 2 : 1;
#pragma unroll 1
            for (int c = 0; c < kChunks / kTaken; c++) {
                p.col0 = ((int64_t)at.n * kBlocksN * 2 + half * kChunks) / kTaken * 32 + c * 32;
                if (p.col0 >= g.cols) break;
                if (g.wide && p.col0 + 32 <= g.cols) finish_wide<EPI>(g, acc[0], acc[kTaken - 1], p, s1, s2, buf, lane);
                else finish_any<EPI>(g, acc[0], acc[kTaken - 1], p, s1, s2, buf, lane);
#pragma unroll
                for (int u = 0; u < kChunks - kTaken; u++)
#pragma unroll
                    for (int i = 0; i < 32; i++) acc[u][i] = acc[u + kTaken][i];
            }
        }
        if (!ok && lane == 0) give_up(g, stop);
        __syncwarp();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    team_sync<CTAS>();  // a pair ends together: each reads and signals the other's memory
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        tmem_free<CTAS>(tmem);
    }
}

template <int CTAS, int PB, bool AMN, bool BMN, int EPI>
__global__ void __launch_bounds__(kGemmThreads, 1) k_gemm(const __grid_constant__ GemmArgs g) {
    multiply<CTAS, PB, AMN, BMN, EPI>(g, (int)blockIdx.x, (int)gridDim.x);
}
// dx and dw of a small layer side by side: `first` blocks for dx, the others for dw (333 x 515 x 257: 22 us the whole call, 32 one
// after the other).
template <int PB>
__global__ void __launch_bounds__(kGemmThreads, 1) k_both(const __grid_constant__ GemmArgs dx, const __grid_constant__ GemmArgs dw, int first) {
    if ((int)blockIdx.x < first) multiply<1, 2, false, true, EPI_STORE>(dx, (int)blockIdx.x, first);
    else multiply<1, PB, true, true, EPI_STORE>(dw, (int)blockIdx.x - first, (int)gridDim.x - first);
}

// ---------------------------------------------------------------- how a product is cut

// Estimated cycles of a way of cutting: rounds of whole tiles, then rounds of slices. A k-block takes a pair 1,750 cycles,
// bound by what the L2 delivers, and a single block, which fetches as much for half the work, the same when most SMs run,
// 1,100 when few do; a tile's first fetches and what of its epilogue nothing covers 9,000 (6,000 single); a slice's sums
// are written once and read once, 3,000 each (1,500); where a kernel of its own reads them,
// a tenth of that, and 8,000 for it to come and go.
static double cut_cost(int ctas, int64_t tiles, int64_t k_blocks, int64_t slices, bool store) {
    const int64_t teams = kPlanSMs / ctas, rounds = tiles / teams, rest = tiles % teams;
    const int64_t busy = rounds > 0 ? kPlanSMs : rest * slices * ctas;
    const double block = ctas == 2 || busy > 100 ? 1750 : 1100, tile = ctas == 2 ? 9000 : 6000, slice = ctas == 2 ? 3000 : 1500;
    double t = (double)rounds * (block * (double)k_blocks + tile);
    if (rest) t += (double)((rest * slices + teams - 1) / teams) * (block * (double)((k_blocks + slices - 1) / slices) + tile);
    if (later(store ? EPI_STORE : EPI_LINEAR, (int)slices)) return t + slice * (1.0 + 0.1 * (double)slices) + 8000;
    return slices > 1 ? t + slice * (double)(1 + slices) : t;
}

GemmPlan gemm_plan(int64_t m_blocks, int64_t n_blocks, int64_t k_blocks, bool store) {
    GemmPlan best{};
    double least = 0;
    for (int ctas = 1; ctas <= 2; ctas++) {
        const int64_t mt = (m_blocks + 2 * ctas - 1) / (2 * ctas), nt = (n_blocks + 2 * ctas - 1) / (2 * ctas), tiles = mt * nt;
        const int64_t teams = kPlanSMs / ctas, rest = tiles % teams;
        for (int64_t s = 1; s <= k_blocks && s <= 16 && (s == 1 || rest * s <= 3 * teams); s++) {
            const double t = cut_cost(ctas, tiles, k_blocks, s, store);
            if (best.ctas && t >= least) continue;
            least = t;
            best.ctas = ctas, best.m_tiles = (int)mt, best.n_tiles = (int)nt;
            best.whole = (int)(s > 1 ? tiles - rest : tiles), best.slices = (int)s;
            best.counters = s > 1 ? (int)rest * ctas * kEpiWarps : 0;
            best.partial_bytes = s > 1 ? (size_t)(rest * s) * (size_t)ctas * 128 * (128 * (size_t)ctas) * sizeof(float) : 0;
        }
    }
    return best;
}

static int unit_count(const GemmPlan& p) { return p.whole + (p.m_tiles * p.n_tiles - p.whole) * p.slices; }
bool side_by_side(const GemmPlan& dx, const GemmPlan& dw) { return dx.ctas == 1 && dw.ctas == 1 && unit_count(dx) + unit_count(dw) <= 2 * kPlanSMs; }

static GemmPlan set_plan(GemmArgs& g, bool gated, bool store) {
    const GemmPlan p = gemm_plan(g.a.mn_blocks, gated ? 2 * (int64_t)g.gate_blocks : g.b.mn_blocks, g.k_blocks, store);
    g.m_tiles = p.m_tiles, g.n_tiles = p.n_tiles, g.whole = p.whole, g.slices = p.slices;
    return p;
}
template <class Kernel>
static cudaError_t allow_shared(Kernel kernel) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes); }
template <int CTAS>
static cudaError_t launch_slices(const GemmArgs& g, cudaStream_t st) {
    const int cut = g.m_tiles * g.n_tiles - g.whole;  // of CTAS x kEpiWarps parts of 8 CTAS eights each
    return launch_early(k_slices<CTAS>, dim3((unsigned)(cut * CTAS * kEpiWarps * 8 * CTAS / (kSliceThreads / 32))), kSliceThreads, 0, st, 1, g);
}
template <int CTAS, int PB, bool AMN, bool BMN, int EPI>
static cudaError_t launch_one(const GemmArgs& g, int units, int sm_count, cudaStream_t st) {
    static const cudaError_t ready = allow_shared(k_gemm<CTAS, PB, AMN, BMN, EPI>);
    if (ready != cudaSuccess) return ready;
    const int teams = sm_count / CTAS;
    const cudaError_t rc = launch_early(k_gemm<CTAS, PB, AMN, BMN, EPI>, dim3((unsigned)(CTAS * (units < teams ? units : teams))), kGemmThreads, kSmemBytes, st, CTAS, g);
    return rc != cudaSuccess || !later(EPI, g.slices) ? rc : launch_slices<CTAS>(g, st);
}
template <int PB, bool AMN, bool BMN, int EPI>
static cudaError_t launch_sized(GemmArgs& g, int sm_count, cudaStream_t st) {
    const GemmPlan p = set_plan(g, EPI == EPI_GATED, EPI == EPI_STORE);
    return p.ctas == 1 ? launch_one<1, PB, AMN, BMN, EPI>(g, unit_count(p), sm_count, st) : launch_one<2, PB, AMN, BMN, EPI>(g, unit_count(p), sm_count, st);
}
template <int PB>
static cudaError_t launch_pair(const GemmArgs& dx, int dx_units, const GemmArgs& dw, int dw_units, cudaStream_t st) {
    static const cudaError_t ready = allow_shared(k_both<PB>);
    if (ready != cudaSuccess) return ready;
    return launch_early(k_both<PB>, dim3((unsigned)(dx_units + dw_units)), kGemmThreads, kSmemBytes, st, 1, dx, dw, dx_units);
}

static bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

static void set_access(GemmArgs& g) {
    const bool ck = g.save8 || g.save8_2;
    g.wide = g.cols % (ck ? 8 : 4) == 0 && aligned(g.out, 16) && aligned(g.out2, 16) && aligned(g.bias, 16) && aligned(g.bias2, 16) &&
             aligned(g.residual, 16) && aligned(g.save, 16) && aligned(g.save2, 16) && aligned(g.save8, 8) && aligned(g.save8_2, 8);
    g.groups = ck8_groups(g.cols), g.exp_offset = ck8_exp_offset(g.rows, g.cols);
}

cudaError_t launch_gemm(const GemmArgs& args, bool a_mn, bool b_mn, int pieces_b, Epilogue epi, int sm_count, cudaStream_t st) {
    GemmArgs g = args;
    set_access(g);
    if (epi == EPI_LINEAR) return launch_sized<2, false, false, EPI_LINEAR>(g, sm_count, st);
    if (epi == EPI_GATED) return launch_sized<2, false, false, EPI_GATED>(g, sm_count, st);
    if (!a_mn && b_mn) return launch_sized<2, false, true, EPI_STORE>(g, sm_count, st);
    if (a_mn && b_mn && pieces_b == 2) return launch_sized<2, true, true, EPI_STORE>(g, sm_count, st);
    if (a_mn && b_mn && pieces_b == 1) return launch_sized<1, true, true, EPI_STORE>(g, sm_count, st);
    return cudaErrorInvalidValue;
}

cudaError_t launch_gemm_pair(const GemmArgs& dx_args, const GemmArgs& dw_args, int pieces_b, cudaStream_t st, int& launches) {
    GemmArgs dx = dx_args, dw = dw_args;
    set_access(dx), set_access(dw);
    const GemmPlan px = set_plan(dx, false, true), pw = set_plan(dw, false, true);
    launches = 1;
    cudaError_t rc = pieces_b == 1 ? launch_pair<1>(dx, unit_count(px), dw, unit_count(pw), st) : launch_pair<2>(dx, unit_count(px), dw, unit_count(pw), st);
    if (rc == cudaSuccess && later(EPI_STORE, dx.slices)) rc = launch_slices<1>(dx, st), launches++;
    if (rc == cudaSuccess && later(EPI_STORE, dw.slices)) rc = launch_slices<1>(dw, st), launches++;
    return rc;
}

}  // namespace slb_ffn
