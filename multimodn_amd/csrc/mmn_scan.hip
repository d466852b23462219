// mmn_scan.hip -- gfx950 kernels and C entry points of the selective scan (include/mmn_sequence.h).
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <initializer_list>

#include "mmn_hip.h"
#include "mmn_sequence.h"

namespace {
typedef float f32x4 __attribute__((ext_vector_type(4)));
#include "seq_common.inc"
#include "seq_sum.inc"
#include "seq_scan.inc"
}  // namespace

#include "seq_host.inc"

// Steps' distance in x, dt, z or dy.  Of one step, or none, it is the width, whatever the caller says: the kernels walk steps in pieces
// and rely on those behind the last lying behind the buffer's end.
static int64_t step_of(const mmn_seq_scan_desc* s, int64_t stride) { return s->steps > 1 ? stride : s->width; }

static int padded_states(int n) { return n <= 4 ? 4 : n <= 8 ? 8 : n <= 16 ? 16 : 32; }

struct ScanPlan {
    int waves, cblocks, seg, nseg, nmark, ck_log2, near, slots;
    int64_t grid;
    bool sorted, order;     // rows' order is made and kept with the marks; it is used
    size_t off_order, off_segh, off_segdt, off_part, off_mid, off_bc, bytes;
};
static ScanPlan scan_plan(const mmn_seq_scan_desc* s, bool backward) {
    ScanPlan p;
    const int per = s->width / s->groups, tiles = (int)ceil_div(per, 64);
    // Waves a workgroup: as few lanes without a channel as there can be, then as few workgroups
    int best = 1 << 30;
    p.waves = 1;
    for (int w = 1; w <= 4; ++w) {
        const int blocks = (int)ceil_div(tiles, w), cost = 4 * blocks * w + blocks;
        if (cost < best) { best = cost; p.waves = w; }
    }
    p.cblocks = (int)ceil_div(tiles, p.waves);
    // Segments, each of which costs a first pass over its steps: enough for two waves on each of the 1024 SIMDs (all that fit of the
    // backward kernel), half as many again where rows differ in length (4 rows of up to 2048 steps, 1024 channels: 241 us forward and
    // backward with three waves a SIMD, 270 with two, 248 with four).  From 896 waves on the rows are enough by themselves (512 steps, 64
    // channels, fp32: 600 rows 790 us in segments and 965 in one piece; 1000 rows 1071 and 1045; 1500 rows 1631 and 1511).
    const int64_t waves = s->batch * s->groups * tiles;
    const int64_t want = waves >= 896 ? 1 : ceil_div(1024 * (s->lengths ? 3 : 2), waves > 0 ? waves : 1);
    // Marks, and so segments, every 8 steps where 16 leave half the SIMDs without a wave (64 channels, 16 states, fp32, forward and
    // backward: 16 rows of 100 steps 44 us instead of 54, 1 row of 1024 48 instead of 60, but 256 rows of 60 72 instead of 63; 1 row of
    // 4096 steps 72 instead of 71, for its link).
    p.ck_log2 = s->steps <= 2048 && waves * ceil_div(s->steps, SCAN_CK) <= 512 ? 3 : 4;
    const int ck = 1 << p.ck_log2;
    int64_t n = ceil_div(s->steps, ck);
    n = want < n ? want : n;
    // ... and as many as it takes for a segment of the widest strided tensor to stay below 2^30 bytes (32-bit offsets in the kernels)
    int64_t stride = s->width;
    for (const int64_t t : {s->x_step, s->dt_step, s->z ? s->z_step : 0, backward ? s->dy_step : 0})
        if (step_of(s, t) > stride) stride = step_of(s, t);
    const int64_t fits = ((int64_t)1 << 30) / (stride * 4) / ck * ck;
    if (fits > 0 && ceil_div(s->steps, fits) > n) n = ceil_div(s->steps, fits);
    p.seg = n > 1 ? (int)(ceil_div(ceil_div(s->steps, n), ck) * ck) : (s->steps > 0 ? s->steps : 1);
    p.nseg = s->steps > 0 ? (int)ceil_div(s->steps, p.seg) : 1;
    // segments join their states themselves (64 rows of 250 steps in 16 segments: 29 us forward, by k_scan_link 26)
    p.near = p.nseg <= (p.ck_log2 == 3 ? 16 : 8);
    p.nmark = (int)ceil_div(s->steps, ck);
    // Backward: rows at a time, the others in turn behind them (8192 waves: eight for each SIMD)
    const int64_t most = 8192 / ((int64_t)s->groups * tiles);
    p.slots = (int)(backward && p.nseg == 1 && s->batch > most ? (most > 0 ? most : 1) : s->batch);
    p.grid = (int64_t)p.slots * p.nseg * s->groups * p.cblocks;
    size_t at = 0;
    auto take = [&](size_t n) { const size_t o = at; at += pad256(n); return o; };
    const size_t rows = (size_t)s->batch * p.nseg, parts = (size_t)p.slots * p.nseg;
    // (4096 rows of up to 48 steps, 64 channels: 46 + 132 us and 5.4 for the order, instead of 58 + 175.  Many rows even out by
    // themselves, one workgroup orders them, and rows taken in turn have to be the same ones in every run.)
    p.sorted = s->lengths && s->steps > 0 && waves >= 896 && s->batch <= 16384;       // (by sizes alone: both passes agree on it)
    p.order = p.sorted && p.nseg == 1 && p.slots == s->batch;
    p.off_order = take(p.order && !s->marks ? sizeof(int32_t) * (size_t)s->batch : 0);
    p.off_segh = take(p.nseg > 1 ? sizeof(float) * rows * s->states * s->width : 0);
    p.off_segdt = take(p.nseg > 1 ? sizeof(float) * rows * s->width : 0);
    p.off_part = p.off_mid = p.off_bc = at;
    if (backward) {
        const int64_t n = (int64_t)(s->states + 2) * s->width;
        p.off_part = take(sizeof(float) * parts * n);
        p.off_mid = take(sum_parts_bytes((int64_t)parts, n));
        p.off_bc = take(p.cblocks > 1 ? sizeof(float) * (size_t)p.cblocks * s->batch * s->steps * s->groups * 2 * s->states : 0);
    }
    p.bytes = at > 0 ? at : 256;
    return p;
}

static bool scan_sizes_ok(const mmn_seq_scan_desc* s) {
    return s && s->batch >= 0 && s->batch <= MAX_GRID && s->steps >= 0 && s->steps <= (1 << 30) && s->width >= 1 && s->groups >= 1 && s->width % s->groups == 0 &&
           s->states >= 1 && s->states <= MMN_SEQ_MAX_STATES && s->type >= 0 && s->type <= 2;
}
// A segment of at least SCAN_CK_FEW steps is addressed with 32-bit offsets; steps that share memory would not read as 0 behind the end
static bool scan_strides_ok(const mmn_seq_scan_desc* s, bool backward) {
    const int64_t most = 1 << 23;
    auto ok = [&](int64_t stride) { return step_of(s, stride) >= s->width && step_of(s, stride) <= most; };
    return s->width <= most && ok(s->x_step) && ok(s->dt_step) && (!s->z || ok(s->z_step)) && (!backward || ok(s->dy_step));
}

template <typename S> static size_t marks_of(const S& s, const ScanPlan& p) { return (size_t)s.batch * p.nmark * s.states * s.width; }

static ScanArgs scan_args(const mmn_seq_scan_desc* s, const ScanPlan& p, char* ws) {
    ScanArgs a;
    a.x = s->x; a.dt = s->dt; a.b = s->b; a.c = s->c; a.z = s->z; a.dy = s->dy;
    a.a = s->a; a.d = s->d; a.dt_bias = s->dt_bias; a.state = s->state; a.dstate_out = s->dstate_out; a.lengths = s->lengths;
    a.y = s->y; a.dx = s->dx; a.ddt = s->ddt; a.dz = s->dz; a.db = s->db; a.dc = s->dc;
    a.state_out = s->state_out; a.dstate = s->dstate;
    // the rows' order lies behind the marks, where a forward pass leaves it for the backward
    a.order = !p.order ? nullptr : s->marks ? (const int32_t*)(s->marks + marks_of(*s, p)) : (const int32_t*)(ws + p.off_order);
    a.seg_h = (float*)(ws + p.off_segh); a.seg_dt = (float*)(ws + p.off_segdt); a.marks = s->marks;
    a.part = (float*)(ws + p.off_part); a.bc_part = (float*)(ws + p.off_bc);
    a.batch = s->batch;
    a.xb = s->x_row; a.xt = step_of(s, s->x_step); a.dtb = s->dt_row; a.dtt = step_of(s, s->dt_step); a.bb = s->b_row; a.bt = s->b_step; a.bg = s->b_group;
    a.cb = s->c_row; a.ct = s->c_step; a.cg = s->c_group; a.zb = s->z_row; a.zt = step_of(s, s->z_step); a.dyb = s->dy_row; a.dyt = step_of(s, s->dy_step);
    a.steps = s->steps; a.width = s->width; a.groups = s->groups; a.states = s->states; a.softplus = s->softplus;
    a.seg = p.seg; a.nseg = p.nseg; a.nmark = p.nmark; a.ck_log2 = p.ck_log2; a.near = p.near; a.cblocks = p.cblocks; a.slots = p.slots;
    return a;
}

template <typename T, int NP>
static int scan_forward(const ScanArgs& a, const ScanPlan& p, hipStream_t st) {
    const dim3 grid((unsigned)p.grid), block(64 * p.waves);
    if (p.sorted && (a.order || a.marks)) {
        int32_t* order = a.order ? const_cast<int32_t*>(a.order) : (int32_t*)(a.marks + marks_of(a, p));
        SEQ_LAUNCH(k_scan_order, dim3(1), dim3(1024), 0, st, a.lengths, order, (int)a.batch, a.steps);
    }
    if (p.nseg > 1) {
        SEQ_LAUNCH((k_scan_part<T, NP, false>), grid, block, 0, st, a);
        const int64_t lanes = a.batch * a.states * a.width;
        if (p.near) {}                                       // (the segments themselves: link_near)
        else if (p.nseg > LINK_U) SEQ_LAUNCH((k_scan_link<false, 4>), dim3((unsigned)ceil_div(lanes, 64)), dim3(256), 0, st, a);
        else SEQ_LAUNCH((k_scan_link<false, 1>), dim3((unsigned)ceil_div(lanes, 256)), dim3(256), 0, st, a);
    }
    if (a.marks) SEQ_LAUNCH((k_scan<T, NP, true>), grid, block, 0, st, a);
    else SEQ_LAUNCH((k_scan<T, NP, false>), grid, block, 0, st, a);
    return MMN_OK;
}

template <typename T, int NP>
static int scan_backward(const ScanArgs& a, const ScanPlan& p, float* mid, float* dparams, hipStream_t st) {
    const dim3 grid((unsigned)p.grid), block(64 * p.waves);
    if (p.nseg > 1) {
        SEQ_LAUNCH((k_scan_part<T, NP, true>), grid, block, 0, st, a);
        const int64_t lanes = a.batch * a.states * a.width;
        if (p.near) {}                                       // (the segments themselves: link_near)
        else if (p.nseg > LINK_U) SEQ_LAUNCH((k_scan_link<true, 4>), dim3((unsigned)ceil_div(lanes, 64)), dim3(256), 0, st, a);
        else SEQ_LAUNCH((k_scan_link<true, 1>), dim3((unsigned)ceil_div(lanes, 256)), dim3(256), 0, st, a);
    }
    const size_t lds = ScanShape<NP>::grad_lds(p.waves);
    const bool many = p.slots < a.batch;
    const hipError_t e = hipFuncSetAttribute(many ? reinterpret_cast<const void*>(k_scan_grad<T, NP, true>) : reinterpret_cast<const void*>(k_scan_grad<T, NP, false>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)ScanShape<NP>::grad_lds(4));
    if (e != hipSuccess) { mmn_note_hip_error((int)e); return MMN_ERR_HIP; }
    if (many) SEQ_LAUNCH((k_scan_grad<T, NP, true>), grid, block, lds, st, a);
    else SEQ_LAUNCH((k_scan_grad<T, NP, false>), grid, block, lds, st, a);
    const float* part = a.part;
    int64_t parts = (int64_t)p.slots * p.nseg;
    const int64_t n = (int64_t)(a.states + 2) * a.width, rows = a.batch * a.steps * a.groups;
    const int rc = sum_many_parts(part, parts, mid, n, a.width, st);
    if (rc != MMN_OK) return rc;
    const int64_t sum_wg = ceil_div(n, SUM_COLS), bc_wg = p.cblocks > 1 ? ceil_div(rows * 2 * a.states, SUM_NT) : 0;
    if (sum_wg + bc_wg > MAX_GRID) return MMN_ERR_UNSUPPORTED;
    SEQ_LAUNCH(k_scan_sums<T>, dim3((unsigned)(sum_wg + bc_wg)), dim3(SUM_NT), 0, st, part, dparams, parts, n, a.width, a.states, (unsigned)sum_wg,
               a.bc_part, (T*)a.db, (T*)a.dc, rows, a.states, p.cblocks);
    return MMN_OK;
}

#define SCAN_STATES(FN, T, ...)                                                                                          \
    (padded_states(s->states) == 4 ? FN<T, 4>(__VA_ARGS__) : padded_states(s->states) == 8 ? FN<T, 8>(__VA_ARGS__)       \
     : padded_states(s->states) == 16 ? FN<T, 16>(__VA_ARGS__) : FN<T, 32>(__VA_ARGS__))
#define SCAN_TYPES(FN, ...)                                                                                              \
    (s->type == MMN_SEQ_F32 ? SCAN_STATES(FN, float, __VA_ARGS__) : s->type == MMN_SEQ_BF16 ? SCAN_STATES(FN, bf16, __VA_ARGS__) : SCAN_STATES(FN, f16, __VA_ARGS__))

extern "C" {

size_t mmn_seq_scan_marks(const mmn_seq_scan_desc* s) {
    if (!scan_sizes_ok(s)) return 0;
    const ScanPlan p = scan_plan(s, false);
    return marks_of(*s, p) + (p.sorted ? (size_t)s->batch : 0);
}

size_t mmn_seq_scan_bytes(const mmn_seq_scan_desc* s, int backward) { return scan_sizes_ok(s) ? scan_plan(s, backward != 0).bytes : 0; }

int mmn_seq_scan(const mmn_seq_scan_desc* s, void* ws, size_t ws_bytes, void* stream) {
    if (!scan_sizes_ok(s)) return MMN_ERR_ARG;
    if (s->batch == 0) return MMN_OK;
    if (!s->a || (s->steps > 0 && (!s->x || !s->dt || !s->b || !s->c || !s->y))) return MMN_ERR_ARG;
    if (!scan_strides_ok(s, false)) return MMN_ERR_UNSUPPORTED;
    const ScanPlan p = scan_plan(s, false);
    if (!ws || !aligned(ws, 256) || ws_bytes < p.bytes) return MMN_ERR_WORKSPACE;
    if (p.grid > MAX_GRID || ceil_div(s->batch * s->states * s->width, 64) > MAX_GRID) return MMN_ERR_UNSUPPORTED;
    const hipStream_t st = (hipStream_t)stream;
    const ScanArgs a = scan_args(s, p, (char*)ws);
    return SCAN_TYPES(scan_forward, a, p, st);
}

int mmn_seq_scan_grad(const mmn_seq_scan_desc* s, void* ws, size_t ws_bytes, void* stream) {
    if (!scan_sizes_ok(s)) return MMN_ERR_ARG;
    if (s->batch == 0 || s->steps == 0) return MMN_ERR_UNSUPPORTED;
    if (!s->a || !s->x || !s->dt || !s->b || !s->c || !s->marks || !s->dy || !s->dx || !s->ddt || !s->db || !s->dc || !s->dparams ||
        (s->z && !s->dz)) return MMN_ERR_ARG;
    if (!scan_strides_ok(s, true)) return MMN_ERR_UNSUPPORTED;
    const ScanPlan p = scan_plan(s, true);
    if (!ws || !aligned(ws, 256) || ws_bytes < p.bytes) return MMN_ERR_WORKSPACE;
    if (p.grid > MAX_GRID || ceil_div(s->batch * s->states * s->width, 64) > MAX_GRID ||
        ceil_div(s->batch * s->steps * s->groups * 2 * s->states, SUM_NT) > MAX_GRID) return MMN_ERR_UNSUPPORTED;
    const hipStream_t st = (hipStream_t)stream;
    const ScanArgs a = scan_args(s, p, (char*)ws);
    return SCAN_TYPES(scan_backward, a, p, (float*)((char*)ws + p.off_mid), s->dparams, st);
}

int mmn_seq_scan_step(const mmn_seq_scan_desc* s, void* stream) {
    if (!scan_sizes_ok(s)) return MMN_ERR_ARG;
    if (s->batch == 0) return MMN_OK;
    if (!s->a || !s->x || !s->dt || !s->b || !s->c || !s->y || !s->state || !s->state_out) return MMN_ERR_ARG;
    const hipStream_t st = (hipStream_t)stream;
    ScanPlan p = {};
    ScanArgs a = scan_args(s, p, nullptr);
    // four states a lane where every channel's begin on 16 bytes
    const bool four = s->states % 4 == 0 && aligned(s->state, 16) && aligned(s->state_out, 16) && aligned(s->a, 16);
    const int q = log2_up(ceil_div(s->states, four ? 4 : 1), 5);
    const int64_t gx = ceil_div((s->batch * s->width) << q, 256);
    if (gx > MAX_GRID) return MMN_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)gx);
    // b and c four at a time too where every row's and group's begin on such a vector
    const size_t vec = 4 * type_size(s->type);
    const int bc = four && aligned(s->b, vec) && aligned(s->c, vec) && s->b_row % 4 == 0 && s->c_row % 4 == 0 && s->b_group % 4 == 0 && s->c_group % 4 == 0;
    // states beyond what the last-level cache (256 MB) holds are not kept there
    const bool past = (double)s->batch * s->width * s->states * sizeof(float) * (s->state == s->state_out ? 1 : 2) > 200e6;
#define STEP(T)                                                                                          \
    do {                                                                                                 \
        if (four && past) SEQ_LAUNCH((k_scan_step<T, 4, true>), grid, dim3(256), 0, st, a, q, bc);       \
        else if (four) SEQ_LAUNCH((k_scan_step<T, 4, false>), grid, dim3(256), 0, st, a, q, bc);         \
        else SEQ_LAUNCH((k_scan_step<T, 1, false>), grid, dim3(256), 0, st, a, q, bc);                   \
    } while (0)
    if (s->type == MMN_SEQ_F32) STEP(float);
    else if (s->type == MMN_SEQ_BF16) STEP(bf16);
    else STEP(f16);
#undef STEP
    return MMN_OK;
}

}  // extern "C"
