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

constexpr int BM = 128;
constexpr int kEpiWarps = 8;
constexpr int kGemmThreads = 128 + 32 * kEpiWarps;          // a warpgroup that copies and issues, two of the epilogue
// Registers: three warpgroups start with 168 a thread, 504 in all; the first keeps 56 and the other two, which hold
// 128 sums a thread, take 224 each: 504 again.
constexpr int kIssueRegs = 56, kEpiRegs = 224;
constexpr int kRingBytes = 192 * 1024;
constexpr int kTurnFloats = 32 * 32;                        // one warp's turning buffer
constexpr int kSmemBytes = kRingBytes + kEpiWarps * kTurnFloats * 4 + 256 + 1024;
constexpr int kSegment = 4;                                 // k-blocks per accumulator segment
constexpr int kMaxStages = 4;
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

// Blocks of B along N in a column of tiles: all, or at its end as many as exist -- an even number, so that a pair can halve
// it (what is not there is never stored).
template <int CTAS, int EPI>
__device__ __forceinline__ int blocks_wide(const GemmArgs& g, int n) {
    const int most = 2 * CTAS;
    const int left = EPI == EPI_GATED ? 2 * (g.gate_blocks - n * (most / 2)) : g.b.mn_blocks - n * most;
    return left >= most ? most : (left + 1) & ~1;
}
// Where chunk c (32 columns) of a warp's half lies in a tile's accumulator. Gated: the first half of the chunks are columns
// of the gate, the others the same columns of the second product, which follow 64 later.
template <int EPI, int CHUNKS>
__device__ __forceinline__ constexpr unsigned column_of(int half, int c) {
    if (EPI != EPI_GATED) return (unsigned)(half * CHUNKS + c) * 32;
    const int j = half * (CHUNKS / 2) + c % (CHUNKS / 2);
    return (unsigned)((j >> 1) * 128 + (j & 1) * 32 + (c >= CHUNKS / 2 ? 64 : 0));
}

// ---------------------------------------------------------------- epilogue

struct Piece {          // rows x 32 columns of the output
    int64_t row0, col0;
    int rows;           // that exist
};

// A warp's 4 KiB turning buffer: 32 rows of 32 columns, or 16 of 64 for the gated pair, in 16-byte chunks whose place
// within a row is exclusive-ored with the row's low bits, so that rows written by their lanes and rows read by eight lanes
// both spread over all banks.
template <int EPI>
__device__ __forceinline__ int turned(int row, int chunk) {
    constexpr int kChunksPerRow = EPI == EPI_GATED ? 16 : 8;
    return (row * kChunksPerRow + (chunk ^ (row & 7))) * 4;
}

// Keeps pre-activations, in fp32, as a checkpoint, or both (null: not), at element `at` of the tensor and exponent byte
// `group` of the checkpoint. Four columns: eight neighbouring lanes hold the group.
__device__ __forceinline__ void keep4(const float4& v, int64_t at, int64_t group, const GemmArgs& g, float* full, char* ck, int lane) {
    if (full) *reinterpret_cast<float4*>(full + at) = v;
    if (ck) {
        unsigned top = max(max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu),
                           max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu));
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(0xffu << (lane & 24), top, o));
        const unsigned byte = ck8_exponent(top);
        *reinterpret_cast<unsigned*>(ck + at) = ck8_quantise4(v.x, v.y, v.z, v.w, byte);
        if ((lane & 7) == 0) ck[g.exp_offset + group] = (char)byte;
    }
}
// One column: the warp holds the group.
__device__ __forceinline__ void keep1(float v, bool ok, int64_t at, int64_t group, const GemmArgs& g, float* full, char* ck, int lane) {
    if (full && ok) full[at] = v;
    if (ck) {
        const unsigned byte = ck8_exponent(__reduce_max_sync(0xffffffffu, ok ? __float_as_uint(v) & 0x7fffffffu : 0u));
        if (ok) ck[at] = (char)ck8_quantise(v, byte);
        if (lane == 0) ck[g.exp_offset + group] = (char)byte;
    }
}
__device__ __forceinline__ float4 scaled(const float* p, float s1, float s2, const float4& bias) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    return make_float4(fmaf(v.x * s1, s2, bias.x), fmaf(v.y * s1, s2, bias.y), fmaf(v.z * s1, s2, bias.z), fmaf(v.w * s1, s2, bias.w));
}

// The rows of a piece out of the turning buffer. Loops of a few rows, not straight code: the epilogue runs once per tile,
// and code of its unrolled length spends its time fetching instructions (150 k cycles a tile). The activation is chosen
// outside them and one offset serves all tensors: what is left is bound by instructions issued, and 128 sums leave few
// registers.
template <int EPI, int ROWS, int ACT>
__device__ __forceinline__ void finish_rows(const GemmArgs& g, const float* buf, const Piece& p, float s1, float s2, int lane) {
    const bool second = EPI == EPI_STORE && p.row0 >= g.split;
    const int64_t first = p.row0 - (second ? g.split : 0);
    float* out = second ? g.out2 : g.out;
    constexpr int kAtOnce = EPI == EPI_LINEAR ? 2 : 4;
    if (g.wide && p.col0 + 32 <= g.cols) {  // 16-byte accesses: eight lanes a row, four rows at a time
        const int chunk = lane & 7;
        const int64_t col = p.col0 + chunk * 4, row = first + (lane >> 3);
        const float4 none = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const float4 bias = EPI != EPI_STORE && g.bias ? __ldg(reinterpret_cast<const float4*>(g.bias + col)) : none;
        const float4 bias2 = EPI == EPI_GATED && g.bias2 ? __ldg(reinterpret_cast<const float4*>(g.bias2 + col)) : none;
        int64_t at = row * g.cols + col, group = EPI == EPI_STORE ? 0 : row * g.groups + col / kGroup;
#pragma unroll 1
        for (int r0 = lane >> 3; r0 < ROWS; r0 += 4 * kAtOnce) {
            float4 add[kAtOnce];
            if (EPI == EPI_LINEAR && g.residual) {
#pragma unroll
                for (int i = 0; i < kAtOnce; i++) add[i] = r0 + 4 * i < p.rows ? *reinterpret_cast<const float4*>(g.residual + at + 4 * i * g.cols) : none;
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; i++) {
                const int r = r0 + 4 * i;
                if (r < p.rows) {  // the same for the eight lanes of a row
                    float4 v = scaled(buf + turned<EPI>(r, chunk), s1, s2, bias);
                    if (EPI != EPI_STORE) {
                        keep4(v, at, group, g, g.save, g.save8, lane);
                        v = make_float4(act_of(ACT, v.x), act_of(ACT, v.y), act_of(ACT, v.z), act_of(ACT, v.w));
                    }
                    if (EPI == EPI_GATED) {
                        const float4 w = scaled(buf + turned<EPI>(r, 8 + chunk), s1, s2, bias2);
                        keep4(w, at, group, g, g.save2, g.save8_2, lane);
                        v = make_float4(v.x * w.x, v.y * w.y, v.z * w.z, v.w * w.w);
                    }
                    if (EPI == EPI_LINEAR && g.residual) v = make_float4(v.x + add[i].x, v.y + add[i].y, v.z + add[i].z, v.w + add[i].w);
                    *reinterpret_cast<float4*>(out + at) = v;
                }
                at += 4 * g.cols, group += 4 * g.groups;
            }
        }
        return;
    }
    const int64_t col = p.col0 + lane;  // any alignment: a column per lane, several rows' loads in flight
    const bool ok = col < g.cols;
    const float bias = EPI != EPI_STORE && g.bias && ok ? __ldg(g.bias + col) : 0.0f;
    const float bias2 = EPI == EPI_GATED && g.bias2 && ok ? __ldg(g.bias2 + col) : 0.0f;
    int64_t at = first * g.cols + col, group = EPI == EPI_STORE ? 0 : first * g.groups + p.col0 / kGroup;
#pragma unroll 1
    for (int r0 = 0; r0 < ROWS && r0 < p.rows; r0 += 2 * kAtOnce) {
        float add[2 * kAtOnce];
        if (EPI == EPI_LINEAR && g.residual) {
#pragma unroll
            for (int i = 0; i < 2 * kAtOnce; i++) add[i] = ok && r0 + i < p.rows ? g.residual[at + i * g.cols] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 2 * kAtOnce; i++) {
            const int r = r0 + i;
            if (r < p.rows) {
                float v = fmaf(buf[turned<EPI>(r, lane >> 2) + (lane & 3)] * s1, s2, bias);
                if (EPI != EPI_STORE) {
                    keep1(v, ok, at, group, g, g.save, g.save8, lane);
                    v = act_of(ACT, v);
                }
                if (EPI == EPI_GATED) {
                    const float w = fmaf(buf[turned<EPI>(r, 8 + (lane >> 2)) + (lane & 3)] * s1, s2, bias2);
                    keep1(w, ok, at, group, g, g.save2, g.save8_2, lane);
                    v *= w;
                }
                if (EPI == EPI_LINEAR && g.residual) v += add[i];
                if (ok) out[at] = v;
            }
            at += g.cols, group += g.groups;
        }
    }
}
template <int EPI, int ROWS>
__device__ __forceinline__ void finish_piece(const GemmArgs& g, const float* buf, const Piece& p, float s1, float s2, int lane) {
    if (EPI == EPI_STORE || g.act == ACT_NONE) finish_rows<EPI, ROWS, ACT_NONE>(g, buf, p, s1, s2, lane);
    else if (g.act == ACT_GELU) finish_rows<EPI, ROWS, ACT_GELU>(g, buf, p, s1, s2, lane);
    else finish_rows<EPI, ROWS, ACT_SILU>(g, buf, p, s1, s2, lane);
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

// CTAS = 1: a block per tile of 128 x 128. CTAS = 2: a pair of blocks (a cluster) per tile of 256 x 256: each holds 128 rows of A
// and 128 columns' worth of B in its shared memory and 128 rows of the accumulator, and the first issues products that
// read both. Per value fetched a pair computes twice as much, which is what bounds large products: fetching from L2.
// Warp 0 copies, warp 1 issues the products (in a pair's second block: reports arrived stages to the first), warps 4 to
// 11 read the accumulators: two per 32 rows, each half the columns.
template <int CTAS, int PB, bool AMN, bool BMN, int EPI>
__global__ void __launch_bounds__(kGemmThreads, 1) k_gemm(const __grid_constant__ GemmArgs g) {
    constexpr int BN = 128 * CTAS, kBlocksN = BN / kBlock, kHalf = BN / 2, kChunks = kHalf / 32;
    constexpr int kOperandBytes = 2 * (int)kImageBytes;  // one piece of this block's 128 rows of A, or of its share of B
    constexpr int kStageBytes = (2 + PB) * kOperandBytes;
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
    const int rank = CTAS == 2 ? (int)(blockIdx.x & 1) : 0;
    const int team = (int)blockIdx.x / CTAS, teams = (int)gridDim.x / CTAS;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; s++) mbar_init(full + 8 * s, 1), mbar_init(empty + 8 * s, 1), mbar_init(peer_full + 8 * s, 1);
        for (int b = 0; b < 2; b++) mbar_init(tfull + 8 * b, 1), mbar_init(tempty + 8 * b, CTAS * kEpiWarps);
        mbar_init(drained, 1);
        *stop = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) tmem_alloc<CTAS>(smem_addr(words + 1));
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    team_sync<CTAS>();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = *reinterpret_cast<volatile unsigned*>(words + 1);
    const int tiles = g.m_tiles * g.n_tiles;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
        if (warp == 0 && lane == 0) {
            unsigned it = 0;
            bool ok = true;
            for (int t = team; ok && t < tiles; t += teams) {
                const Tile at = tile_at(t, g.m_tiles, g.n_tiles);
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
                const unsigned bytes = (unsigned)(na * 2 + nb * PB) * (unsigned)kImageBytes;
                for (int kb = 0; kb < g.k_blocks; kb++, it++) {
                    const unsigned s = it % kStages, round = it / kStages;
                    if (!mbar_wait(empty + 8 * s, (round & 1) ^ 1, g.timeout_ns, stop)) {
                        ok = false;
                        break;
                    }
                    const unsigned bar = full + 8 * s, at_a = ring_at + s * kStageBytes, at_b = at_a + 2 * kOperandBytes;
                    mbar_expect(bar, bytes);
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        if (i >= na) break;
                        const char* src = g.a.plane + ((int64_t)(ma + i) * g.a.mn_stride + (int64_t)kb * g.a.k_stride) * (int64_t)(2 * kImageBytes);
                        bulk_load(at_a + i * kImageBytes, src, kImageBytes, bar);
                        bulk_load(at_a + kOperandBytes + i * kImageBytes, src + kImageBytes, kImageBytes, bar);
                    }
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        if (j >= nb) break;
                        const char* src = g.b.plane + (b_at[j] + (int64_t)kb * g.b.k_stride) * (int64_t)(PB * kImageBytes);
                        bulk_load(at_b + j * kImageBytes, src, kImageBytes, bar);
                        if (PB == 2) bulk_load(at_b + kOperandBytes + j * kImageBytes, src + kImageBytes, kImageBytes, bar);
                    }
                }
            }
            if (!ok) {  // nothing may still be on its way into this block's shared memory when it ends
                give_up(g, stop);
                for (unsigned back = it < (unsigned)kStages ? it : (unsigned)kStages; back > 0; back--) {
                    const unsigned i = it - back;
                    mbar_wait(full + 8 * (i % kStages), (i / kStages) & 1, g.timeout_ns, nullptr);
                }
            }
        }
        if (warp == 1 && lane == 0 && rank == 0) {
            unsigned it = 0, seg = 0;
            bool ok = true;
            for (int t = team; ok && t < tiles; t += teams) {
                const Tile at = tile_at(t, g.m_tiles, g.n_tiles);
                const unsigned idesc = 1u << 4 | (AMN ? 1u << 15 : 0u) | (BMN ? 1u << 16 : 0u) | (unsigned)(blocks_wide<CTAS, EPI>(g, at.n) * kBlock >> 3) << 17 |
                                       (unsigned)(BM * CTAS >> 4) << 24;
                for (int k0 = 0; ok && k0 < g.k_blocks; k0 += kSegment, seg++) {
                    const unsigned buf = seg & 1, d = tmem + buf * BN;
                    if (!mbar_wait<CTAS == 2>(tempty + 8 * buf, ((seg >> 1) & 1) ^ 1, g.timeout_ns, stop)) {
                        ok = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const int k1 = min(k0 + kSegment, g.k_blocks);
                    for (int kb = k0; kb < k1; kb++, it++) {
                        const unsigned s = it % kStages;
                        if (!mbar_wait(full + 8 * s, (it / kStages) & 1, g.timeout_ns, stop) ||
                            (CTAS == 2 && !mbar_wait<true>(peer_full + 8 * s, (it / kStages) & 1, g.timeout_ns, stop))) {
                            ok = false;
                            break;
                        }
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const unsigned at_a = ring_at + s * kStageBytes, at_b = at_a + 2 * kOperandBytes;
#pragma unroll
                        for (int product = 0; product < 1 + PB; product++) {  // hi*hi, lo*hi, hi*lo
                            const uint64_t da = descriptor<AMN>(at_a + (product == 1 ? kOperandBytes : 0));
                            const uint64_t db = descriptor<BMN>(at_b + (product == 2 ? kOperandBytes : 0));
#pragma unroll
                            for (int step = 0; step < kBlock / 16; step++)
                                mma_f16<CTAS>(d, da + (uint64_t)(step * kStepBytes<AMN> >> 4), db + (uint64_t)(step * kStepBytes<BMN> >> 4), idesc,
                                              !(kb == k0 && product == 0 && step == 0));
                        }
                        mma_commit<CTAS>(empty + 8 * s);
                    }
                    if (ok) mma_commit<CTAS>(tfull + 8 * buf);
                }
            }
            if (!ok) {
                give_up(g, stop);
                mma_commit<CTAS>(drained);
                mbar_wait(drained, 0, g.timeout_ns, nullptr);
            }
        }
        if (CTAS == 2 && warp == 1 && lane == 0 && rank == 1) {
            const unsigned there = remote(peer_full, 0);
            const int rounds = tiles > team ? ((tiles - team - 1) / teams + 1) * g.k_blocks : 0;
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
        const int e = g.exps[g.a.exp_id] + g.exps[g.b.exp_id] - 30;  // undo both planes' scaling, in two steps that cannot overflow early
        const float s1 = exp2f((float)(e / 2)), s2 = exp2f((float)(e - e / 2));
        unsigned seg = 0;
        bool ok = true;
        for (int t = team; ok && t < tiles; t += teams) {
            const Tile at = tile_at(t, g.m_tiles, g.n_tiles);
            float acc[kChunks][32];
#pragma unroll
            for (int c = 0; c < kChunks; c++)
#pragma unroll
                for (int i = 0; i < 32; i++) acc[c][i] = 0.0f;
            if (EPI == EPI_LINEAR && g.residual) {  // into L2 while the products run: a lane a row, this warp's columns
                const int64_t row = (int64_t)(at.m * CTAS + rank) * BM + q * 32 + lane, col = (int64_t)at.n * BN + half * kHalf;
                if (row < g.rows)
                    for (int64_t c = col; c < min(col + kHalf, g.cols); c += 32)
                        asm volatile("prefetch.global.L2 [%0];" ::"l"(g.residual + row * g.cols + c));
            }
            for (int k0 = 0; k0 < g.k_blocks; k0 += kSegment, seg++) {
                const unsigned b = seg & 1;
                ok = __all_sync(0xffffffffu, mbar_wait(tfull + 8 * b, (seg >> 1) & 1, g.timeout_ns, stop));
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                for (int c = 0; c < kChunks; c++) {
                    float v[32];
                    tmem_load32(tmem + ((unsigned)(q * 32) << 16) + b * BN + column_of<EPI, kChunks>(half, c), v);
#pragma unroll
                    for (int i = 0; i < 32; i++) acc[c][i] += v[i];
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    if (CTAS == 1) mbar_arrive(tempty + 8 * b);
                    else mbar_arrive_remote_relaxed(remote(tempty + 8 * b, 0));  // only reads of tensor memory go before it, and those are complete
                }
            }
            if (!ok) break;
            Piece p;
            p.row0 = (int64_t)(at.m * CTAS + rank) * BM + q * 32;
            int64_t left = g.rows - p.row0;
            if (EPI == EPI_STORE && p.row0 >= g.split) left += g.split;
            p.rows = left < 0 ? 0 : left < 32 ? (int)left : 32;
            if (p.rows == 0) continue;
            const int all_rows = p.rows;
            const int64_t row0 = p.row0;
#pragma unroll 1
            for (int c = 0; c < (EPI == EPI_GATED ? kChunks / 2 : kChunks); c++) {
                p.col0 = EPI == EPI_GATED ? (int64_t)at.n * kHalf + (half * (kChunks / 2) + c) * 32 : (int64_t)at.n * BN + half * kHalf + c * 32;
                if (p.col0 >= g.cols) break;
                if (EPI == EPI_GATED) {
#pragma unroll 1
                    for (int pass = 0; pass < 2; pass++) {  // 16 rows of both at a time fit the buffer
                        __syncwarp();
                        if (lane >> 4 == pass) {
#pragma unroll
                            for (int u = 0; u < kChunks / 2; u++)
                                if (c == u)
#pragma unroll
                                    for (int i = 0; i < 16; i++) {
                                        const float* from = i < 8 ? acc[u] + 4 * i : acc[u + kChunks / 2] + 4 * (i - 8);
                                        *reinterpret_cast<float4*>(buf + turned<EPI>(lane & 15, i)) = make_float4(from[0], from[1], from[2], from[3]);
                                    }
                        }
                        __syncwarp();
                        p.row0 = row0 + 16 * pass, p.rows = min(16, all_rows - 16 * pass);
                        finish_piece<EPI, 16>(g, buf, p, s1, s2, lane);
                    }
                } else {
                    __syncwarp();
#pragma unroll
                    for (int u = 0; u < kChunks; u++)
                        if (c == u)
#pragma unroll
                            for (int i = 0; i < 8; i++)
                                *reinterpret_cast<float4*>(buf + turned<EPI>(lane, i)) =
                                    make_float4(acc[u][4 * i], acc[u][4 * i + 1], acc[u][4 * i + 2], acc[u][4 * i + 3]);
                    __syncwarp();
                    finish_piece<EPI, 32>(g, buf, p, s1, s2, lane);
                }
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
static cudaError_t launch_one(GemmArgs g, int sm_count, cudaStream_t st) {
    static const cudaError_t ready = cudaFuncSetAttribute(k_gemm<CTAS, PB, AMN, BMN, EPI>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    if (ready != cudaSuccess) return ready;
    const int width = EPI == EPI_GATED ? 2 * g.gate_blocks : g.b.mn_blocks;
    g.m_tiles = (g.a.mn_blocks + 2 * CTAS - 1) / (2 * CTAS), g.n_tiles = (width + 2 * CTAS - 1) / (2 * CTAS);
    const int tiles = g.m_tiles * g.n_tiles, teams = sm_count / CTAS;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(CTAS * (tiles < teams ? tiles : teams))), cfg.blockDim = dim3(kGemmThreads);
    cfg.dynamicSmemBytes = kSmemBytes, cfg.stream = st;
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = CTAS, cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    cfg.attrs = &cluster, cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_gemm<CTAS, PB, AMN, BMN, EPI>, g);
}
template <int PB, bool AMN, bool BMN, int EPI>
static cudaError_t launch_sized(const GemmArgs& g, int sm_count, cudaStream_t st) {
    // Single blocks as long as their smaller tiles all run at once: a pair's tile would take longer. Beyond that the
    // pairs' smaller traffic decides.
    const int64_t width = EPI == EPI_GATED ? 2 * (int64_t)g.gate_blocks : g.b.mn_blocks;
    const int64_t singles = ((g.a.mn_blocks + 1) / 2) * ((width + 1) / 2);
    return singles <= sm_count ? launch_one<1, PB, AMN, BMN, EPI>(g, sm_count, st) : launch_one<2, PB, AMN, BMN, EPI>(g, sm_count, st);
}

static bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

cudaError_t launch_gemm(const GemmArgs& args, bool a_mn, bool b_mn, int pieces_b, Epilogue epi, int sm_count, cudaStream_t st) {
    GemmArgs g = args;
    g.wide = g.cols % 4 == 0 && aligned(g.out, 16) && aligned(g.out2, 16) && aligned(g.bias, 16) && aligned(g.bias2, 16) && aligned(g.residual, 16) &&
             aligned(g.save, 16) && aligned(g.save2, 16) && aligned(g.save8, 4) && aligned(g.save8_2, 4);
    g.groups = ck8_groups(g.cols), g.exp_offset = ck8_exp_offset(g.rows, g.cols);
    if (epi == EPI_LINEAR) return launch_sized<2, false, false, EPI_LINEAR>(g, sm_count, st);
    if (epi == EPI_GATED) return launch_sized<2, false, false, EPI_GATED>(g, sm_count, st);
    if (!a_mn && b_mn) return launch_sized<2, false, true, EPI_STORE>(g, sm_count, st);
    if (a_mn && b_mn && pieces_b == 2) return launch_sized<2, true, true, EPI_STORE>(g, sm_count, st);
    if (a_mn && b_mn && pieces_b == 1) return launch_sized<1, true, true, EPI_STORE>(g, sm_count, st);
    return cudaErrorInvalidValue;
}

}  // namespace slb_ffn
