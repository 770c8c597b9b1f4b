// Entry points of the feed-forward operators and of the 8-bit checkpoints (include/soliton_b200.h): argument checks,
// the layout of their scratch, and the order of their launches. Two levels, like the rest of the library: `slb_linear`
// and its like take their scratch from the pool, on meta as on cuda, so that a dry run plans it; `slb_cuda_linear` and
// its like are for a host core that owns the allocator and passes the scratch in.
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/soliton_b200.h"
#include "dp_engine.hpp"
#include "ffn.hpp"
#include "pool.hpp"

using namespace slb;
using namespace slb_ffn;

namespace {

constexpr int64_t kMostExtent = int64_t(1) << 30;  // rows and columns: block and tile counts stay within 32 bits
constexpr int64_t kMostBlocks = int64_t(1) << 30;

int64_t blocks_of(int64_t n) { return (n + kBlock - 1) / kBlock; }
size_t round_up(size_t n) { return (n + 1023) & ~size_t(1023); }

bool extents_ok(int64_t m, int64_t n, int64_t k) {
    return m >= 0 && n >= 1 && k >= 1 && m <= kMostExtent && n <= kMostExtent && k <= kMostExtent && blocks_of(m) * blocks_of(n) <= kMostBlocks &&
           blocks_of(m) * blocks_of(k) <= kMostBlocks && blocks_of(n) * blocks_of(k) <= kMostBlocks;
}
bool act_ok(int act) { return act == ACT_NONE || act == ACT_GELU || act == ACT_SILU; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

// The scratch of a call, laid out front to back; with base = nullptr only counted.
struct Carver {
    char* base;
    size_t used = 0;
    char* take(size_t n) {
        char* p = base ? base + used : nullptr;
        used += round_up(n);
        return p;
    }
};
struct Scratch {
    int *exps, *guess;
    unsigned* tops;
    float *parts, *colsum, *colsum2;
    float *row_factor, *col_factor, *col_factor2;
    char *y, *x, *w;        // planes: the gradient of the pre-activations, the input, the weights
    float* partial;
    int* counters;          // of the first product, then of the second
    int n_counters;
};
// weights: one, or the gated block's two side by side (each padded to whole blocks)
size_t carve(Scratch& s, void* base, int64_t m, int64_t n, int64_t k, int weights, bool backward) {
    Carver c{static_cast<char*>(base)};
    s = Scratch{};
    const int64_t mb = blocks_of(m), nb = blocks_of(n), kb = blocks_of(k);
    const size_t block = 2 * kImageBytes;
    size_t partial;
    s.x = c.take((size_t)(mb * kb) * block);
    s.w = c.take((size_t)(weights * nb * kb) * block);
    if (backward) {
        const GemmPlan dx = gemm_plan(mb, kb, weights * nb, true), dw = gemm_plan(weights * nb, kb, mb, true), half = gemm_plan(nb, kb, mb, true);
        const int dw_counters = dw.counters > half.counters ? dw.counters : half.counters;
        s.y = c.take((size_t)(weights * mb * nb) * block);
        s.exps = reinterpret_cast<int*>(c.take(kMaxPlanes * sizeof(int)));
        s.guess = reinterpret_cast<int*>(c.take(kMaxPlanes * sizeof(int)));
        s.tops = reinterpret_cast<unsigned*>(c.take(kMaxPlanes * sizeof(unsigned)));
        s.parts = reinterpret_cast<float*>(c.take(kMaxSlots * kAmaxParts * sizeof(float)));
        s.colsum = reinterpret_cast<float*>(c.take((size_t)(mb * n) * sizeof(float)));
        s.colsum2 = weights == 2 ? reinterpret_cast<float*>(c.take((size_t)(mb * n) * sizeof(float))) : nullptr;
        s.n_counters = dx.counters + dw_counters;
        partial = side_by_side(dx, dw) ? dx.partial_bytes + dw.partial_bytes : dx.partial_bytes > dw.partial_bytes ? dx.partial_bytes : dw.partial_bytes;
        if (half.partial_bytes > partial) partial = half.partial_bytes;  // one of the gated pair's weights alone
    } else {
        const GemmPlan p = gemm_plan(mb, weights * nb, kb, false);
        s.row_factor = reinterpret_cast<float*>(c.take((size_t)(mb * kBlock) * sizeof(float)));
        s.col_factor = reinterpret_cast<float*>(c.take((size_t)(nb * kBlock) * sizeof(float)));
        s.col_factor2 = weights == 2 ? reinterpret_cast<float*>(c.take((size_t)(nb * kBlock) * sizeof(float))) : nullptr;
        s.n_counters = p.counters, partial = p.partial_bytes;
    }
    s.counters = reinterpret_cast<int*>(c.take((size_t)s.n_counters * sizeof(int)));
    s.partial = reinterpret_cast<float*>(c.take(partial));
    return c.used;
}

// A call on the library's device: what the optimizer path has recorded goes out first, lanes that still work on a
// tensor are waited for, launches are counted.
class Op {
public:
    Op() : e_(Engine::get()) {
        if (!e_.cuda_ready()) {
            e_.set_error(ERR_NO_WORKSPACE);
            return;
        }
        if (cudaGetDevice(&before_) != cudaSuccess || (before_ != e_.ordinal() && cudaSetDevice(e_.ordinal()) != cudaSuccess)) {
            e_.set_error(ERR_LAUNCH);
            return;
        }
        e_.flush();
        ok = true;
    }
    ~Op() {
        if (before_ >= 0 && before_ != e_.ordinal() && e_.cuda_ready()) cudaSetDevice(before_);
    }
    void reads(const void* p, int64_t bytes) {
        if (p && bytes > 0) e_.legacy_touches(p, (size_t)bytes, false);
    }
    void writes(void* p, int64_t bytes) {
        if (p && bytes > 0) e_.legacy_touches(p, (size_t)bytes, true);
    }
    void launched(cudaError_t rc, int count = 1) {
        if (rc != cudaSuccess) failed_ = true;
        count_ += count;
    }
    int done() {
        e_.legacy_launches(count_);
        if (failed_) e_.set_error(ERR_LAUNCH);
        return failed_ ? -1 : 0;
    }
    int sms() const { return e_.sm_count(); }
    int* status() const { return e_.status_word(); }
    unsigned long long timeout_ns() const { return e_.opt.timeout_ns; }
    bool ok = false;

private:
    Engine& e_;
    int before_ = -1, count_ = 0;
    bool failed_ = false;
};

int refuse(int code) {
    Engine::get().set_error(code);
    return -1;
}

// ---------------------------------------------------------------- maxima and planes of a call

struct Planner {
    PackArgs p{};
    explicit Planner(const Scratch& s) {
        p.amax.parts = s.parts, p.amax.tops = s.tops, p.guess = s.guess, p.exps = s.exps, p.counters = s.counters, p.n_counters = s.n_counters;
    }
    int slot(const float* x, const void* ck, int64_t rows, int64_t cols) {
        AmaxSlot& t = p.amax.slot[p.amax.slots];
        t.is_ck8 = x == nullptr;
        t.p = x ? static_cast<const void*>(x) : static_cast<const char*>(ck) + ck8_exp_offset(rows, cols);
        t.n = x ? rows * cols : rows * ck8_groups(cols);
        const int64_t want = (t.n * (x ? 4 : 1) + 16383) / 16384;
        t.parts = (int)(want < 1 ? 1 : want < kAmaxParts ? want : kAmaxParts);
        if (x) bytes_ += 4 * t.n;
        return p.amax.slots++;
    }
    PackJob& job(int kind, int64_t rows, int64_t cols, char* plane, int plane_id, int pieces) {
        PackJob& j = p.job[p.jobs++];
        j.kind = kind, j.rows = rows, j.cols = cols;
        j.row_blocks = (int)blocks_of(rows), j.col_blocks = (int)blocks_of(cols), j.row_stride = j.col_blocks;
        j.plane = plane, j.plane_id = plane_id, j.pieces = pieces;
        j.first_unit = p.units;
        p.units += j.row_blocks * j.col_blocks;
        p.planes |= 1 << plane_id;
        return j;
    }
    // the matrix itself, or its checkpoint
    PackJob& matrix(const float* x, const void* ck, int64_t rows, int64_t cols, char* plane, int plane_id, int slots) {
        PackJob& j = job(x ? PACK_FP32 : PACK_CK8, rows, cols, plane, plane_id, x ? 2 : 1);
        j.a = x, j.b8 = x ? nullptr : ck, j.slots = slots;
        return j;
    }
    void launch(Op& op) {
        // Tensors that a second read would find in L2 are read whole; of more, those of 16 MiB up are sampled.
        for (int s = 0; s < p.amax.slots && bytes_ > kReadTwice; s++) {
            AmaxSlot& t = p.amax.slot[s];
            t.sampled = !t.is_ck8 && t.n >= (int64_t(1) << 22);
            p.sampled |= t.sampled;
        }
        op.launched(launch_amax(p.amax, op.sms(), 0));
        op.launched(launch_pack(p, op.sms(), 0));
        if (p.sampled) op.launched(launch_repack(p, op.sms(), 0));
    }

private:
    static constexpr int64_t kReadTwice = int64_t(100) << 20;
    int64_t bytes_ = 0;
};

// Planes of a forward pass.
struct RowPlanner {
    RowArgs r{};
    explicit RowPlanner(const Scratch& s) { r.counters = s.counters, r.n_counters = s.n_counters; }
    void matrix(const float* x, int64_t rows, int64_t cols, char* plane, float* factor, bool is_a) {
        RowJob& j = r.job[r.jobs++];
        j.a = x, j.rows = rows, j.cols = cols, j.col_blocks = (int)blocks_of(cols), j.plane = plane, j.factor = factor, j.is_a = is_a;
        j.first_group = r.groups;
        r.groups += (int)blocks_of(rows) * (kBlock / 8);
    }
};

GemmArgs product(const Op& op, const Scratch& s) {
    GemmArgs g{};
    g.exps = s.exps, g.row_factor = s.row_factor, g.col_factor = s.col_factor, g.col_factor2 = s.col_factor2;
    g.partial = s.partial, g.counters = s.counters, g.status = op.status(), g.timeout_ns = op.timeout_ns(), g.split = INT64_MAX;
    return g;
}
// A plane whose block rows run along M or N (K-major), or along K (MN-major).
Operand k_major(const char* plane, int64_t rows, int64_t row_stride, int exp_id) { return Operand{plane, row_stride, 1, (int)rows, exp_id}; }
Operand mn_major(const char* plane, int64_t cols, int64_t row_stride, int exp_id) { return Operand{plane, 1, row_stride, (int)cols, exp_id}; }

enum { PLANE_Y = 0, PLANE_X = 1, PLANE_W = 2 };

// ---------------------------------------------------------------- the two operators, forward and backward

int run_linear(const float* x, const float* w, const float* bias, const float* residual, float* y, float* pre, void* pre8, int64_t m, int64_t n, int64_t k,
               int act, void* scratch) {
    Op op;
    if (!op.ok) return -1;
    Scratch s;
    const size_t bytes = carve(s, scratch, m, n, k, 1, false);
    op.reads(x, 4 * m * k), op.reads(w, 4 * n * k), op.reads(bias, 4 * n), op.reads(residual, 4 * m * n);
    op.writes(y, 4 * m * n), op.writes(pre, 4 * m * n), op.writes(pre8, pre8 ? ck8_bytes(m, n) : 0), op.writes(scratch, (int64_t)bytes);
    RowPlanner p(s);
    p.matrix(x, m, k, s.x, s.row_factor, true), p.matrix(w, n, k, s.w, s.col_factor, false);
    op.launched(launch_rows(p.r, 0));
    GemmArgs g = product(op, s);
    const int64_t kb = blocks_of(k);
    g.a = k_major(s.x, blocks_of(m), kb, PLANE_X), g.b = k_major(s.w, blocks_of(n), kb, PLANE_W);
    g.k_blocks = (int)kb, g.k_len = k, g.rows = m, g.cols = n, g.act = act;
    g.out = y, g.bias = bias, g.residual = residual, g.save = pre, g.save8 = static_cast<char*>(pre8);
    op.launched(launch_gemm(g, false, false, 2, EPI_LINEAR, op.sms(), 0));
    return op.done();
}

int run_gated(const float* x, const float* wg, const float* wu, const float* bg, const float* bu, float* h, float* gate, float* up, void* gate8, void* up8,
              int64_t m, int64_t f, int64_t k, int act, void* scratch) {
    Op op;
    if (!op.ok) return -1;
    Scratch s;
    const size_t bytes = carve(s, scratch, m, f, k, 2, false);
    op.reads(x, 4 * m * k), op.reads(wg, 4 * f * k), op.reads(wu, 4 * f * k), op.reads(bg, 4 * f), op.reads(bu, 4 * f);
    op.writes(h, 4 * m * f), op.writes(gate, 4 * m * f), op.writes(up, 4 * m * f), op.writes(scratch, (int64_t)bytes);
    op.writes(gate8, gate8 ? ck8_bytes(m, f) : 0), op.writes(up8, up8 ? ck8_bytes(m, f) : 0);
    const int64_t kb = blocks_of(k), fb = blocks_of(f);
    RowPlanner p(s);
    p.matrix(x, m, k, s.x, s.row_factor, true), p.matrix(wg, f, k, s.w, s.col_factor, false);
    p.matrix(wu, f, k, s.w + fb * kb * (int64_t)(2 * kImageBytes), s.col_factor2, false);
    op.launched(launch_rows(p.r, 0));
    GemmArgs g = product(op, s);
    g.a = k_major(s.x, blocks_of(m), kb, PLANE_X), g.b = k_major(s.w, 2 * fb, kb, PLANE_W);
    g.k_blocks = (int)kb, g.k_len = k, g.rows = m, g.cols = f, g.act = act, g.gate_blocks = (int)fb;
    g.out = h, g.bias = bg, g.bias2 = bu, g.save = gate, g.save2 = up, g.save8 = static_cast<char*>(gate8), g.save8_2 = static_cast<char*>(up8);
    op.launched(launch_gemm(g, false, false, 2, EPI_GATED, op.sms(), 0));
    return op.done();
}

// What the two backward passes share: dx = dY W and dW = dY^T x over the planes, with dY and W of both gated halves side
// by side (`width` blocks in all).
void gradients(Op& op, const Scratch& s, bool x_ck8, float* dx, float* dw, float* dw2, int64_t m, int64_t n, int64_t k, int halves) {
    const int64_t mb = blocks_of(m), nb = blocks_of(n), kb = blocks_of(k), width = halves * nb;
    const GemmPlan dx_plan = gemm_plan(mb, kb, width, true);
    const bool both = dw && dw2, whole = halves == 1 || both;  // or one of the gated pair alone: its half of the plane
    GemmArgs x = product(op, s), w = product(op, s);
    x.a = k_major(s.y, mb, width, PLANE_Y), x.b = mn_major(s.w, kb, kb, PLANE_W);
    x.k_blocks = (int)width, x.k_len = halves == 2 ? width * kBlock : n, x.rows = m, x.cols = k, x.out = dx;
    w.counters += dx_plan.counters;
    w.a = mn_major(s.y + (whole || dw ? 0 : nb * (int64_t)(2 * kImageBytes)), whole ? width : nb, width, PLANE_Y), w.b = mn_major(s.x, kb, kb, PLANE_X);
    w.k_blocks = (int)mb, w.k_len = m, w.rows = n, w.cols = k, w.out = dw ? dw : dw2;
    if (both) w.split = nb * kBlock, w.out2 = dw2;
    const int pieces = x_ck8 ? 1 : 2;
    if (dx && (dw || dw2) && whole && side_by_side(dx_plan, gemm_plan(width, kb, mb, true))) {
        w.partial += dx_plan.partial_bytes / sizeof(float);
        int launches = 0;
        const cudaError_t rc = launch_gemm_pair(x, w, pieces, 0, launches);
        op.launched(rc, launches);
        return;
    }
    if (dx) op.launched(launch_gemm(x, false, true, 2, EPI_STORE, op.sms(), 0));
    if (dw || dw2) op.launched(launch_gemm(w, true, true, pieces, EPI_STORE, op.sms(), 0));
}
void no_rows(Op& op, float* p, int64_t count) {  // a sum over no rows
    if (p) op.launched(cudaMemsetAsync(p, 0, (size_t)count * 4, 0));
}

int run_linear_bwd(const float* dy, const float* x, const void* x8, const float* w, const float* pre, const void* pre8, float* dx, float* dw, float* db,
                   int64_t m, int64_t n, int64_t k, int act, void* scratch) {
    Op op;
    if (!op.ok) return -1;
    op.writes(dx, 4 * m * k), op.writes(dw, 4 * n * k), op.writes(db, 4 * n);
    if (m == 0) {
        no_rows(op, dw, n * k), no_rows(op, db, n);
        return op.done();
    }
    Scratch s;
    const size_t bytes = carve(s, scratch, m, n, k, 1, true);
    op.reads(dy, 4 * m * n), op.reads(x, 4 * m * k), op.reads(x8, x8 ? ck8_bytes(m, k) : 0), op.reads(w, 4 * n * k);
    op.reads(pre, 4 * m * n), op.reads(pre8, pre8 ? ck8_bytes(m, n) : 0), op.writes(scratch, (int64_t)bytes);
    Planner p(s);
    p.slot(dy, nullptr, m, n);
    PackJob& j = p.job(act == ACT_NONE ? PACK_FP32 : PACK_ACT, m, n, s.y, PLANE_Y, 2);
    j.a = dy, j.b = pre, j.b8 = pre8, j.act = act, j.slots = 1, j.colsum = db ? s.colsum : nullptr;
    if (dw) {
        const int i = p.slot(x, x8, m, k);
        p.matrix(x, x8, m, k, s.x, PLANE_X, 1 << i);
    }
    if (dx) {
        const int i = p.slot(w, nullptr, n, k);
        p.matrix(w, nullptr, n, k, s.w, PLANE_W, 1 << i);
    }
    p.launch(op);
    if (db) op.launched(launch_colsum(s.colsum, db, nullptr, nullptr, (int)blocks_of(m), n, 0));
    gradients(op, s, x8 != nullptr, dx, dw, nullptr, m, n, k, 1);
    return op.done();
}

int run_gated_bwd(const float* dh, const float* x, const void* x8, const float* wg, const float* wu, const float* gate, const float* up, const void* gate8,
                  const void* up8, float* dx, float* dwg, float* dwu, float* dbg, float* dbu, int64_t m, int64_t f, int64_t k, int act, void* scratch) {
    Op op;
    if (!op.ok) return -1;
    op.writes(dx, 4 * m * k), op.writes(dwg, 4 * f * k), op.writes(dwu, 4 * f * k), op.writes(dbg, 4 * f), op.writes(dbu, 4 * f);
    if (m == 0) {
        no_rows(op, dwg, f * k), no_rows(op, dwu, f * k), no_rows(op, dbg, f), no_rows(op, dbu, f);
        return op.done();
    }
    Scratch s;
    const size_t bytes = carve(s, scratch, m, f, k, 2, true);
    op.reads(dh, 4 * m * f), op.reads(x, 4 * m * k), op.reads(x8, x8 ? ck8_bytes(m, k) : 0), op.reads(wg, 4 * f * k), op.reads(wu, 4 * f * k);
    op.reads(gate, 4 * m * f), op.reads(up, 4 * m * f), op.reads(gate8, gate8 ? ck8_bytes(m, f) : 0), op.reads(up8, up8 ? ck8_bytes(m, f) : 0);
    op.writes(scratch, (int64_t)bytes);
    const int64_t fb = blocks_of(f), kb = blocks_of(k);
    Planner p(s);
    p.slot(dh, nullptr, m, f), p.slot(up, up8, m, f), p.slot(gate, gate8, m, f);  // in the order k_pack bounds the products
    PackJob& j = p.job(PACK_GATED, m, f, s.y, PLANE_Y, 2);
    j.a = dh, j.b = gate, j.b8 = gate8, j.c = up, j.c8 = up8, j.act = act;
    j.row_stride = (int)(2 * fb), j.second = (int)fb;
    j.colsum = dbg ? s.colsum : nullptr, j.colsum2 = dbu ? s.colsum2 : nullptr;
    if (dwg || dwu) {
        const int i = p.slot(x, x8, m, k);
        p.matrix(x, x8, m, k, s.x, PLANE_X, 1 << i);
    }
    if (dx) {
        const int i = p.slot(wg, nullptr, f, k);
        p.slot(wu, nullptr, f, k);
        p.matrix(wg, nullptr, f, k, s.w, PLANE_W, 3 << i);
        p.matrix(wu, nullptr, f, k, s.w + fb * kb * (int64_t)(2 * kImageBytes), PLANE_W, 3 << i);
    }
    p.launch(op);
    if (dbg || dbu) op.launched(launch_colsum(s.colsum, dbg, s.colsum2, dbu, (int)blocks_of(m), f, 0));
    gradients(op, s, x8 != nullptr, dx, dwg, dwu, m, f, k, 2);
    return op.done();
}

// ---------------------------------------------------------------- argument checks

bool linear_ok(const float* x, const float* w, const float* bias, const float* residual, const float* y, const float* pre, int64_t m) {
    return m == 0 || (x && w && y && aligned4(x) && aligned4(w) && aligned4(bias) && aligned4(residual) && aligned4(y) && aligned4(pre));
}
bool one_of(const void* a, const void* b) { return (a != nullptr) != (b != nullptr); }

bool linear_bwd_ok(const float* dy, const float* x, const void* x8, const float* w, const float* pre, const void* pre8, const float* dx, const float* dw,
                   const float* db, int64_t m, int act) {
    if (!dx && !dw && !db) return false;
    if (!aligned4(dx) || !aligned4(dw) || !aligned4(db)) return false;
    if (m == 0) return true;
    if (!dy || !aligned4(dy) || (dx && !w) || !aligned4(w) || (dw && !one_of(x, x8)) || !aligned4(x) || !aligned4(pre)) return false;
    return act == ACT_NONE || one_of(pre, pre8);
}
bool gated_ok(const float* x, const float* wg, const float* wu, const float* bg, const float* bu, const float* h, const float* gate, const float* up, int64_t m) {
    return m == 0 || (x && wg && wu && h && aligned4(x) && aligned4(wg) && aligned4(wu) && aligned4(bg) && aligned4(bu) && aligned4(h) && aligned4(gate) && aligned4(up));
}
bool gated_bwd_ok(const float* dh, const float* x, const void* x8, const float* wg, const float* wu, const float* gate, const float* up, const void* gate8,
                  const void* up8, const float* dx, const float* dwg, const float* dwu, const float* dbg, const float* dbu, int64_t m) {
    if (!dx && !dwg && !dwu && !dbg && !dbu) return false;
    if (!aligned4(dx) || !aligned4(dwg) || !aligned4(dwu) || !aligned4(dbg) || !aligned4(dbu)) return false;
    if (m == 0) return true;
    if (!dh || !aligned4(dh) || (dx && (!wg || !wu)) || !aligned4(wg) || !aligned4(wu) || ((dwg || dwu) && !one_of(x, x8)) || !aligned4(x)) return false;
    return one_of(gate, gate8) && one_of(up, up8) && aligned4(gate) && aligned4(up);
}

// Scratch from the pool for the length of `body`: taken and given back on meta as on cuda.
template <class Body>
int with_scratch(int dev, int64_t m, int64_t n, int64_t k, int weights, bool backward, Body body) {
    if (m == 0) return dev == DEV_CUDA ? body(nullptr) : 0;
    Scratch s;
    const size_t bytes = carve(s, nullptr, m, n, k, weights, backward);
    if (dev == DEV_CUDA && !Engine::get().cuda_ready()) return refuse(ERR_NO_WORKSPACE);
    void* p = pool(dev).alloc(bytes);
    if (!p) return -2;
    const int rc = dev == DEV_CUDA ? body(p) : 0;
    pool(dev).release(p, bytes);  // the next owner's work on it comes later on the same stream
    return rc;
}
// 0: go on; otherwise the code to return. `sizes` and `pointers`: whether they are acceptable.
int admit(int dev, bool sizes, bool pointers) {
    if (!valid_dev(dev)) return -1;
    if (dev == DEV_CPU) return refuse(ERR_NO_CPU_COMPUTE);
    return sizes && (dev == DEV_META || pointers) ? 0 : refuse(ERR_BAD_ARG);
}
// The backend level's: scratch that is large enough and aligned as its layout needs.
bool scratch_ok(const void* p, size_t have, int64_t m, size_t need) { return m == 0 || (p && have >= need && (reinterpret_cast<uintptr_t>(p) & 255) == 0); }

}  // namespace

extern "C" {

size_t slb_linear_scratch_bytes(int64_t m, int64_t n, int64_t k, int backward) {
    Scratch s;
    return extents_ok(m, n, k) && m > 0 ? carve(s, nullptr, m, n, k, 1, backward != 0) : 0;
}
size_t slb_gated_scratch_bytes(int64_t m, int64_t f, int64_t k, int backward) {
    Scratch s;
    return extents_ok(m, f, k) && m > 0 ? carve(s, nullptr, m, f, k, 2, backward != 0) : 0;
}

int slb_cuda_linear(const float* x, const float* w, const float* bias, const float* residual, float* y, float* pre, void* pre8, int64_t m, int64_t n, int64_t k,
                    int act, void* scratch, size_t scratch_bytes) {
    if (!extents_ok(m, n, k) || !act_ok(act) || !linear_ok(x, w, bias, residual, y, pre, m)) return refuse(ERR_BAD_ARG);
    if (m == 0) return 0;
    if (!scratch_ok(scratch, scratch_bytes, m, slb_linear_scratch_bytes(m, n, k, 0))) return refuse(ERR_BAD_ARG);
    return run_linear(x, w, bias, residual, y, pre, pre8, m, n, k, act, scratch);
}
int slb_linear(int dev, const float* x, const float* w, const float* bias, const float* residual, float* y, float* pre, void* pre8, int64_t m, int64_t n,
               int64_t k, int act) {
    const int rc = admit(dev, extents_ok(m, n, k) && act_ok(act), linear_ok(x, w, bias, residual, y, pre, m));
    if (rc != 0 || m == 0) return rc;
    return with_scratch(dev, m, n, k, 1, false, [&](void* s) { return run_linear(x, w, bias, residual, y, pre, pre8, m, n, k, act, s); });
}

int slb_cuda_linear_bwd(const float* dy, const float* x, const void* x8, const float* w, const float* pre, const void* pre8, float* dx, float* dw, float* db,
                        int64_t m, int64_t n, int64_t k, int act, void* scratch, size_t scratch_bytes) {
    if (!extents_ok(m, n, k) || !act_ok(act) || !linear_bwd_ok(dy, x, x8, w, pre, pre8, dx, dw, db, m, act) ||
        !scratch_ok(scratch, scratch_bytes, m, slb_linear_scratch_bytes(m, n, k, 1)))
        return refuse(ERR_BAD_ARG);
    return run_linear_bwd(dy, x, x8, w, pre, pre8, dx, dw, db, m, n, k, act, scratch);
}
int slb_linear_bwd(int dev, const float* dy, const float* x, const void* x8, const float* w, const float* pre, const void* pre8, float* dx, float* dw,
                   float* db, int64_t m, int64_t n, int64_t k, int act) {
    const int rc = admit(dev, extents_ok(m, n, k) && act_ok(act), linear_bwd_ok(dy, x, x8, w, pre, pre8, dx, dw, db, m, act));
    if (rc != 0) return rc;
    return with_scratch(dev, m, n, k, 1, true, [&](void* s) { return run_linear_bwd(dy, x, x8, w, pre, pre8, dx, dw, db, m, n, k, act, s); });
}

int slb_cuda_gated(const float* x, const float* wg, const float* wu, const float* bg, const float* bu, float* h, float* g, float* u, void* g8, void* u8,
                   int64_t m, int64_t f, int64_t k, int act, void* scratch, size_t scratch_bytes) {
    if (!extents_ok(m, f, k) || !act_ok(act) || !gated_ok(x, wg, wu, bg, bu, h, g, u, m)) return refuse(ERR_BAD_ARG);
    if (m == 0) return 0;
    if (!scratch_ok(scratch, scratch_bytes, m, slb_gated_scratch_bytes(m, f, k, 0))) return refuse(ERR_BAD_ARG);
    return run_gated(x, wg, wu, bg, bu, h, g, u, g8, u8, m, f, k, act, scratch);
}
int slb_gated(int dev, const float* x, const float* wg, const float* wu, const float* bg, const float* bu, float* h, float* g, float* u, void* g8, void* u8,
              int64_t m, int64_t f, int64_t k, int act) {
    const int rc = admit(dev, extents_ok(m, f, k) && act_ok(act), gated_ok(x, wg, wu, bg, bu, h, g, u, m));
    if (rc != 0 || m == 0) return rc;
    return with_scratch(dev, m, f, k, 2, false, [&](void* s) { return run_gated(x, wg, wu, bg, bu, h, g, u, g8, u8, m, f, k, act, s); });
}

int slb_cuda_gated_bwd(const float* dh, const float* x, const void* x8, const float* wg, const float* wu, const float* g, const float* u, const void* g8,
                       const void* u8, float* dx, float* dwg, float* dwu, float* dbg, float* dbu, int64_t m, int64_t f, int64_t k, int act, void* scratch,
                       size_t scratch_bytes) {
    if (!extents_ok(m, f, k) || !act_ok(act) || !gated_bwd_ok(dh, x, x8, wg, wu, g, u, g8, u8, dx, dwg, dwu, dbg, dbu, m) ||
        !scratch_ok(scratch, scratch_bytes, m, slb_gated_scratch_bytes(m, f, k, 1)))
        return refuse(ERR_BAD_ARG);
    return run_gated_bwd(dh, x, x8, wg, wu, g, u, g8, u8, dx, dwg, dwu, dbg, dbu, m, f, k, act, scratch);
}
int slb_gated_bwd(int dev, const float* dh, const float* x, const void* x8, const float* wg, const float* wu, const float* g, const float* u, const void* g8,
                  const void* u8, float* dx, float* dwg, float* dwu, float* dbg, float* dbu, int64_t m, int64_t f, int64_t k, int act) {
    const int rc = admit(dev, extents_ok(m, f, k) && act_ok(act), gated_bwd_ok(dh, x, x8, wg, wu, g, u, g8, u8, dx, dwg, dwu, dbg, dbu, m));
    if (rc != 0) return rc;
    return with_scratch(dev, m, f, k, 2, true,
                        [&](void* s) { return run_gated_bwd(dh, x, x8, wg, wu, g, u, g8, u8, dx, dwg, dwu, dbg, dbu, m, f, k, act, s); });
}

// ---------------------------------------------------------------- checkpoints

static bool ck8_extents_ok(int64_t rows, int64_t cols) {
    return rows >= 0 && cols >= 1 && rows <= (int64_t(1) << 40) && cols <= kMostExtent && (rows == 0 || cols <= (int64_t(1) << 40) / rows);
}
size_t slb_ck8_bytes(int64_t rows, int64_t cols) { return ck8_extents_ok(rows, cols) ? (size_t)ck8_bytes(rows, cols) : 0; }

int slb_ck8_save(int dev, const float* x, void* ck, int64_t rows, int64_t cols) {
    const int rc = admit(dev, ck8_extents_ok(rows, cols), rows == 0 || (x && ck && aligned4(x)));
    if (rc != 0 || dev == DEV_META || rows == 0) return rc;
    Op op;
    if (!op.ok) return -1;
    op.reads(x, 4 * rows * cols), op.writes(ck, ck8_bytes(rows, cols));
    op.launched(launch_ck8_save(x, static_cast<char*>(ck), rows, cols, 0));
    return op.done();
}
int slb_ck8_load(int dev, const void* ck, float* x, int64_t rows, int64_t cols) {
    const int rc = admit(dev, ck8_extents_ok(rows, cols), rows == 0 || (x && ck && aligned4(x)));
    if (rc != 0 || dev == DEV_META || rows == 0) return rc;
    Op op;
    if (!op.ok) return -1;
    op.reads(ck, ck8_bytes(rows, cols)), op.writes(x, 4 * rows * cols);
    op.launched(launch_ck8_load(static_cast<const char*>(ck), x, rows, cols, 0));
    return op.done();
}
int slb_ck8_gelu_bwd(int dev, const void* ck, const float* dy, float* dx, int64_t rows, int64_t cols) {
    const int rc = admit(dev, ck8_extents_ok(rows, cols), rows == 0 || (ck && dy && dx && aligned4(dy) && aligned4(dx)));
    if (rc != 0 || dev == DEV_META || rows == 0) return rc;
    Op op;
    if (!op.ok) return -1;
    op.reads(ck, ck8_bytes(rows, cols)), op.reads(dy, 4 * rows * cols), op.writes(dx, 4 * rows * cols);
    op.launched(launch_ck8_gelu_bwd(static_cast<const char*>(ck), dy, dx, rows, cols, 0));
    return op.done();
}

}  // extern "C"
