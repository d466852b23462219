// mmn_sequence.hip -- gfx950 kernels and C entry points of the embedding and convolution operators (include/mmn_sequence.h); the
// selective scan is in mmn_scan.hip.  A translation unit of its own: nothing here shares code with the chain kernels.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>

#include "mmn_hip.h"
#include "mmn_sequence.h"

namespace {
#include "seq_common.inc"
#include "seq_embed.inc"
#include "seq_conv.inc"
#include "seq_sum.inc"
#include "seq_input.inc"
}  // namespace

#include "seq_host.inc"

#ifndef MMN_SOURCE_HASH
#define MMN_SOURCE_HASH "unknown"
#endif
extern "C" const char* mmn_source_hash(void) { return MMN_SOURCE_HASH; }

extern "C" {

// ------------------------------------------------------------------------------------------------ embedding
int mmn_seq_embed(const void* ids, int ids64, const void* table, void* out, int64_t rows, int64_t vocab, int width, int type, float scale, void* stream) {
    if (rows < 0 || rows > MAX_GRID || vocab < 1 || width < 1 || type < 0 || type > 2) return MMN_ERR_ARG;
    if (rows == 0) return MMN_OK;
    const int size = type_size(type);
    if (!ids || !table || !out || !aligned(table, size) || !aligned(out, size) || !aligned(ids, ids64 ? 8 : 4)) return MMN_ERR_ARG;
    const hipStream_t st = (hipStream_t)stream;
    // 16-byte vectors where every row begins on one, else 4-byte ones, else single elements
    const int v = width % (16 / size) == 0 && aligned(table, 16) && aligned(out, 16) ? 16 / size
                : width % (4 / size) == 0 && aligned(table, 4) && aligned(out, 4) ? 4 / size : 1;
    const int l = log2_up(ceil_div(width, v), 6);
    const dim3 grid((unsigned)ceil_div(rows, (256 >> l) * 4));
#define EMBED(T, V)                                                                                                             \
    do {                                                                                                                        \
        if (ids64) SEQ_LAUNCH((k_embed<T, int64_t, V>), grid, dim3(256), 0, st, (const int64_t*)ids, (const T*)table, (T*)out, rows, vocab, width, l, scale); \
        else SEQ_LAUNCH((k_embed<T, int32_t, V>), grid, dim3(256), 0, st, (const int32_t*)ids, (const T*)table, (T*)out, rows, vocab, width, l, scale); \
    } while (0)
    if (type == MMN_SEQ_F32) { if (v == 4) EMBED(float, 4); else EMBED(float, 1); }
    else if (type == MMN_SEQ_BF16) { if (v == 8) EMBED(bf16, 8); else if (v == 2) EMBED(bf16, 2); else EMBED(bf16, 1); }
    else { if (v == 8) EMBED(f16, 8); else if (v == 2) EMBED(f16, 2); else EMBED(f16, 1); }
#undef EMBED
    return MMN_OK;
}

struct EmbedGradPlan {
    int passes, bits, bins, nwg, run, chunk, nchunk, v, ctiles;
    size_t off_hist, off_present, off_keys[2], off_pos[2], off_part, bytes;
};
// `v`: elements a lane sums (the partial sums' size does not depend on it)
static EmbedGradPlan embed_grad_plan(int64_t rows, int64_t vocab, int width) {
    EmbedGradPlan p;
    int need = 1;                                        // bits of the keys 0 .. vocab
    while (((int64_t)1 << need) <= vocab) ++need;
    p.passes = (need + 8) / 9;                           // at most 2^9 bins a pass
    p.bits = (need + p.passes - 1) / p.passes;
    p.bins = 1 << p.bits;
    // Workgroups of whole tiles, at most 128: each reads all counts of all of them.
    const int64_t tiles = ceil_div(rows, SORT_TILE);
    const int64_t per = ceil_div(tiles, 128);
    p.run = (int)(per * SORT_TILE);
    p.nwg = (int)ceil_div(rows, p.run);
    // Entries a chunk: 16 where there are few (more waves), up to 512 (fewer borders to join: 65536 places cost 16 us there with 16)
    int c = 16;
    while (c < 512 && rows / c > 2048) c *= 2;
    p.chunk = c;
    p.nchunk = (int)ceil_div(rows, c);
    size_t at = 0;
    auto take = [&](size_t n) { const size_t o = at; at += pad256(n); return o; };
    p.off_hist = take(sizeof(unsigned) * (size_t)p.nwg * p.bins);
    p.off_present = take(sizeof(unsigned) * (size_t)vocab);
    for (int i = 0; i < 2; ++i) {
        p.off_keys[i] = take(sizeof(unsigned) * (size_t)rows);
        p.off_pos[i] = take(sizeof(unsigned) * (size_t)rows);
    }
    p.off_part = take(sizeof(float) * (size_t)p.nchunk * 2 * width);
    p.bytes = at;
    return p;
}

size_t mmn_seq_embed_grad_bytes(int64_t rows, int64_t vocab, int width) {
    if (rows < 0 || rows > MAX_GRID || vocab < 1 || vocab >= MAX_GRID || width < 1) return 0;
    return embed_grad_plan(rows > 0 ? rows : 1, vocab, width).bytes;
}

int mmn_seq_embed_grad(const void* ids, int ids64, const void* grad, void* out, int64_t rows, int64_t vocab, int width, int type, float scale,
                       void* ws, size_t ws_bytes, void* stream) {
    if (rows < 0 || rows > MAX_GRID || vocab < 1 || vocab >= MAX_GRID || width < 1 || type < 0 || type > 2) return MMN_ERR_ARG;
    const int size = type_size(type);
    if (!out || !aligned(out, size) || (rows > 0 && (!ids || !grad || !aligned(grad, size) || !aligned(ids, ids64 ? 8 : 4)))) return MMN_ERR_ARG;
    const EmbedGradPlan p = embed_grad_plan(rows > 0 ? rows : 1, vocab, width);
    if (!ws || !aligned(ws, 256) || ws_bytes < p.bytes) return MMN_ERR_WORKSPACE;
    const hipStream_t st = (hipStream_t)stream;
    char* w = (char*)ws;
    unsigned* hist = (unsigned*)(w + p.off_hist);
    unsigned* present = (unsigned*)(w + p.off_present);
    unsigned *keys[2], *pos[2];
    for (int i = 0; i < 2; ++i) { keys[i] = (unsigned*)(w + p.off_keys[i]); pos[i] = (unsigned*)(w + p.off_pos[i]); }
    float* part = (float*)(w + p.off_part);
    const int v = width % (16 / size) == 0 && aligned(grad, 16) && aligned(out, 16) ? 16 / size
                : width % (4 / size) == 0 && aligned(grad, 4) && aligned(out, 4) ? 4 / size : 1;
    // A workgroup of k_embed_few has 256 bytes of its table rows.  It is taken where two workgroups a CU own the table (8192 ids, fp32 rows
    // of 203: 12 us instead of 27 for a table of 1501 rows, 18 instead of 30 for 8192, 31 and 31 for 16384; where all 8192 ids are
    // one 36 instead of 19, for its workgroups read them alone).
    const int fv = size == 2 && width % 2 == 0 && aligned(grad, 4) && aligned(out, 4) ? 2 : 1;
    const int64_t tiles = ceil_div(width, 64 * fv);
    if (rows <= FEW_ROWS && vocab * tiles <= 512 * FEW_R) {
        int nb = 0, bits = 0;
        while (((int64_t)1 << nb) < vocab && ((tiles << (nb + 1)) <= 512 || ceil_div(vocab, 1 << nb) > FEW_R)) ++nb;
        while (((int64_t)1 << bits) < ceil_div(vocab, 1 << nb)) ++bits;
        const dim3 fg((unsigned)(tiles << nb));
#define FEW(T, V)                                                                                                                \
    do {                                                                                                                         \
        if (ids64) SEQ_LAUNCH((k_embed_few<T, int64_t, V>), fg, dim3(FEW_NT), 0, st, (const int64_t*)ids, (const T*)grad, (T*)out, (int)rows, (int)vocab, width, (int)tiles, nb, bits, scale); \
        else SEQ_LAUNCH((k_embed_few<T, int32_t, V>), fg, dim3(FEW_NT), 0, st, (const int32_t*)ids, (const T*)grad, (T*)out, (int)rows, (int)vocab, width, (int)tiles, nb, bits, scale); \
    } while (0)
        if (type == MMN_SEQ_F32) FEW(float, 1);
        else if (type == MMN_SEQ_BF16) { if (fv == 2) FEW(bf16, 2); else FEW(bf16, 1); }
        else { if (fv == 2) FEW(f16, 2); else FEW(f16, 1); }
#undef FEW
        return MMN_OK;
    }
    const int nwg = rows > 0 ? p.nwg : 0;
    const bool small = rows > 0 && rows <= SMALL_ROWS && vocab * width <= rows * 16384;   // (a large table is cleared where no id names it only)
    const int64_t clear_wg = ceil_div(vocab, SORT_NT * 8) < 256 ? ceil_div(vocab, SORT_NT * 8) : 256;
    const dim3 hg((unsigned)(nwg + clear_wg)), nt(SORT_NT);
    if (small) {
        const int64_t bytes = vocab * width * size, wg = ceil_div(bytes, 16 * SMALL_NT * 4);
        const dim3 sg(1 + (unsigned)(wg < 1024 ? wg : 1024));
        if (ids64) SEQ_LAUNCH(k_sort_small<int64_t>, sg, dim3(SMALL_NT), 0, st, (const int64_t*)ids, keys[0], pos[0], (int)rows, (int)vocab, p.bits, p.passes, (char*)out, bytes);
        else SEQ_LAUNCH(k_sort_small<int32_t>, sg, dim3(SMALL_NT), 0, st, (const int32_t*)ids, keys[0], pos[0], (int)rows, (int)vocab, p.bits, p.passes, (char*)out, bytes);
    } else if (ids64) SEQ_LAUNCH((k_sort_hist<int64_t, true>), hg, nt, 0, st, (const int64_t*)ids, nullptr, rows, (int)vocab, p.run, nwg, p.bins, 0, hist, present, vocab);
    else SEQ_LAUNCH((k_sort_hist<int32_t, true>), hg, nt, 0, st, (const int32_t*)ids, nullptr, rows, (int)vocab, p.run, nwg, p.bins, 0, hist, present, vocab);
    int at = 0;
    for (int i = 0; i < p.passes && rows > 0 && !small; ++i) {
        if (i == 0) {
            if (ids64) SEQ_LAUNCH((k_sort_pass<int64_t, true>), dim3(nwg), nt, 0, st, (const int64_t*)ids, nullptr, nullptr, keys[0], pos[0], rows, (int)vocab, p.run, p.nwg, p.bits, 0, hist, present);
            else SEQ_LAUNCH((k_sort_pass<int32_t, true>), dim3(nwg), nt, 0, st, (const int32_t*)ids, nullptr, nullptr, keys[0], pos[0], rows, (int)vocab, p.run, p.nwg, p.bits, 0, hist, present);
        } else {
            SEQ_LAUNCH((k_sort_hist<int64_t, false>), dim3(nwg), nt, 0, st, nullptr, keys[at], rows, (int)vocab, p.run, nwg, p.bins, i * p.bits, hist, nullptr, (int64_t)0);
            SEQ_LAUNCH((k_sort_pass<int64_t, false>), dim3(nwg), nt, 0, st, nullptr, keys[at], pos[at], keys[1 - at], pos[1 - at], rows, (int)vocab, p.run, p.nwg, p.bits, i * p.bits, hist, nullptr);
            at = 1 - at;
        }
    }
    const int ctiles = (int)ceil_div(width, 64 * v), nchunk = rows > 0 ? p.nchunk : 0;
    const int64_t sumwg = ceil_div((int64_t)nchunk * ctiles, 4);
    const int64_t zero_wg = small ? 0 : ceil_div(vocab, 16) < 2048 ? ceil_div(vocab, 16) : 2048;
    if (sumwg + zero_wg > MAX_GRID || ceil_div(width, 64) > 65535) return MMN_ERR_UNSUPPORTED;
    const dim3 sg((unsigned)(sumwg + zero_wg));
    const bool join4 = width % 4 == 0 && aligned(out, 4 * size);      // (part begins on 256 bytes)
#define SUM(T, V)                                                                                                                \
    do {                                                                                                                         \
        SEQ_LAUNCH((k_embed_sum<T, V>), sg, dim3(256), 0, st, keys[at], pos[at], (const T*)grad, (T*)out, part, present, rows, (int)vocab, width, p.chunk, nchunk, ctiles, sumwg, scale); \
        if (nchunk > 1 && join4) SEQ_LAUNCH((k_embed_join<T, 4>), dim3((unsigned)ceil_div(nchunk, JOIN_WAVES), (unsigned)ceil_div(width, 256)), dim3(64 * JOIN_WAVES), 0, st, keys[at], part, (T*)out, rows, (int)vocab, width, p.chunk, nchunk, scale); \
        else if (nchunk > 1) SEQ_LAUNCH((k_embed_join<T, 1>), dim3((unsigned)ceil_div(nchunk, JOIN_WAVES), (unsigned)ceil_div(width, 64)), dim3(64 * JOIN_WAVES), 0, st, keys[at], part, (T*)out, rows, (int)vocab, width, p.chunk, nchunk, scale); \
    } while (0)
    if (type == MMN_SEQ_F32) { if (v == 4) SUM(float, 4); else SUM(float, 1); }
    else if (type == MMN_SEQ_BF16) { if (v == 8) SUM(bf16, 8); else if (v == 2) SUM(bf16, 2); else SUM(bf16, 1); }
    else { if (v == 8) SUM(f16, 8); else if (v == 2) SUM(f16, 2); else SUM(f16, 1); }
#undef SUM
    return MMN_OK;
}

// ------------------------------------------------------------------------------------------------ convolution
static bool conv_args(const mmn_seq_conv_desc* c, ConvArgs& a) {
    a.x = c->x; a.dy = c->dy; a.state = c->state; a.dstate_out = c->dstate_out;
    a.y = c->y; a.dx = c->dx; a.state_out = c->state_out; a.dstate = c->dstate;
    a.w = c->weight; a.bias = c->bias; a.lengths = c->lengths; a.part = nullptr;
    a.batch = c->batch; a.xb = c->x_row; a.xt = c->x_step; a.dyb = c->dy_row; a.dyt = c->dy_step;
    a.steps = c->steps; a.width = c->width; a.silu = c->silu;
    a.tiles = (int)ceil_div(c->steps, CONV_RUN);
    return c->batch >= 0 && c->steps >= 0 && c->steps <= (1 << 30) && c->width >= 1 && c->taps >= 2 && c->taps <= 4 && c->type >= 0 && c->type <= 2 &&
           c->batch <= MAX_GRID;
}
// elements a thread takes together: all rows of all tensors begin on such a vector
static int conv_vec(const mmn_seq_conv_desc* c) {
    const int size = type_size(c->type);
    auto fits = [&](int v) {
        const void* ptr[] = {c->x, c->state, c->y, c->state_out, c->dy, c->dstate_out, c->dx, c->dstate};
        for (const void* q : ptr) if (!aligned(q, (size_t)v * size)) return false;
        return c->width % v == 0 && c->x_row % v == 0 && c->x_step % v == 0 && c->dy_row % v == 0 && c->dy_step % v == 0;
    };
    return fits(4) ? 4 : 1;                              // (8 of 16 bits: 22.5 us instead of 18 for 8 x 2048 x 1024 ragged, fewer waves)
}
#define CONV_TAPS(KERN, T, V, ...)                                                   \
    do {                                                                             \
        if (c->taps == 2) SEQ_LAUNCH((KERN<T, V, 2>), __VA_ARGS__);                  \
        else if (c->taps == 3) SEQ_LAUNCH((KERN<T, V, 3>), __VA_ARGS__);             \
        else SEQ_LAUNCH((KERN<T, V, 4>), __VA_ARGS__);                               \
    } while (0)
#define CONV_TYPES(KERN, ...)                                                        \
    do {                                                                             \
        if (c->type == MMN_SEQ_F32) { if (v == 4) CONV_TAPS(KERN, float, 4, __VA_ARGS__); else CONV_TAPS(KERN, float, 1, __VA_ARGS__); } \
        else if (c->type == MMN_SEQ_BF16) { if (v == 4) CONV_TAPS(KERN, bf16, 4, __VA_ARGS__); else CONV_TAPS(KERN, bf16, 1, __VA_ARGS__); } \
        else { if (v == 4) CONV_TAPS(KERN, f16, 4, __VA_ARGS__); else CONV_TAPS(KERN, f16, 1, __VA_ARGS__); } \
    } while (0)

int mmn_seq_conv(const mmn_seq_conv_desc* c, void* stream) {
    ConvArgs a;
    if (!c || !conv_args(c, a)) return MMN_ERR_ARG;
    if (c->batch == 0) return MMN_OK;
    if (!c->weight || (c->steps > 0 && (!c->x || !c->y))) return MMN_ERR_ARG;
    a.tiles = c->steps > 0 ? (int)ceil_div(c->steps, CONV_AHEAD) : 1;      // (no steps: the state still goes on)
    const hipStream_t st = (hipStream_t)stream;
    const int v = conv_vec(c);
    a.lanes_log2 = log2_up(ceil_div(c->width, v), 6);
    const int64_t gx = ceil_div(c->batch * a.tiles, 256 >> a.lanes_log2), gy = ceil_div(ceil_div(c->width, v), 1 << a.lanes_log2);
    if (gx * gy > MAX_GRID) return MMN_ERR_UNSUPPORTED;
    a.cblocks = (int)gy;
    const dim3 grid((unsigned)(gx * gy));
    CONV_TYPES(k_conv, grid, dim3(256), 0, st, a);
    return MMN_OK;
}

struct ConvGradPlan { int v, lanes_log2, parts, gy; int64_t n; size_t off_mid, bytes; };
static ConvGradPlan conv_grad_plan(const mmn_seq_conv_desc* c) {
    ConvGradPlan p;
    p.v = conv_vec(c);
    p.lanes_log2 = log2_up(ceil_div(c->width, p.v), 6);
    p.gy = (int)ceil_div(ceil_div(c->width, p.v), 1 << p.lanes_log2);
    const int64_t jobs = c->batch * ceil_div(c->steps, CONV_RUN), wg = ceil_div(jobs, 256 >> p.lanes_log2);
    const int64_t most = p.gy >= 1024 ? 1 : 1024 / p.gy;  // four workgroups a compute unit; each leaves a partial sum
    p.parts = (int)(wg < 1 ? 1 : wg < most ? wg : most);
    p.n = (int64_t)(c->taps + 1) * c->width;
    p.off_mid = pad256(sizeof(float) * (size_t)p.n * p.parts);
    p.bytes = p.off_mid + sum_parts_bytes(p.parts, p.n);
    return p;
}
size_t mmn_seq_conv_grad_bytes(const mmn_seq_conv_desc* c) {
    ConvArgs a;
    if (!c || !conv_args(c, a)) return 0;
    mmn_seq_conv_desc d = *c;                            // (the largest over all alignments: the vector width decides how many parts there are)
    size_t most = 0;
    const size_t one = conv_grad_plan(&d).bytes;
    d.x_row |= 1;
    const size_t two = conv_grad_plan(&d).bytes;
    most = one > two ? one : two;
    return most;
}
int mmn_seq_conv_grad(const mmn_seq_conv_desc* c, void* ws, size_t ws_bytes, void* stream) {
    ConvArgs a;
    if (!c || !conv_args(c, a)) return MMN_ERR_ARG;
    if (!c->weight || !c->dweight || c->dbias != c->dweight + (int64_t)c->width * c->taps ||
        (c->batch > 0 && c->steps > 0 && (!c->x || !c->dy || !c->dx))) return MMN_ERR_ARG;
    if (c->steps == 0 && c->batch > 0) return MMN_ERR_UNSUPPORTED;
    const ConvGradPlan p = conv_grad_plan(c);
    if (!ws || !aligned(ws, 256) || ws_bytes < p.bytes) return MMN_ERR_WORKSPACE;
    const hipStream_t st = (hipStream_t)stream;
    const int v = p.v;
    a.lanes_log2 = p.lanes_log2;
    a.parts = p.parts;
    a.part = (float*)ws;
    a.cblocks = p.gy;
    const dim3 grid((unsigned)p.parts * p.gy);
    CONV_TYPES(k_conv_grad, grid, dim3(256), 0, st, a);
    return sum_parts(a.part, (float*)((char*)ws + p.off_mid), c->dweight, p.parts, p.n, c->width, c->taps, st);
}

int mmn_seq_conv_step(const mmn_seq_conv_desc* c, void* stream) {
    ConvArgs a;
    if (!c || !conv_args(c, a)) return MMN_ERR_ARG;
    if (c->batch == 0) return MMN_OK;
    if (!c->weight || !c->x || !c->y || !c->state || !c->state_out) return MMN_ERR_ARG;
    const hipStream_t st = (hipStream_t)stream;
    const int v = conv_vec(c);
    a.lanes_log2 = log2_up(ceil_div(c->width, v), 6);
    const int64_t gx = ceil_div(c->batch, CONV_ROWS * (256 >> a.lanes_log2)), gy = ceil_div(ceil_div(c->width, v), 1 << a.lanes_log2);
    if (gx * gy > MAX_GRID) return MMN_ERR_UNSUPPORTED;
    a.cblocks = (int)gy;
    const dim3 grid((unsigned)(gx * gy));
    CONV_TYPES(k_conv_step, grid, dim3(256), 0, st, a);
    return MMN_OK;
}

int mmn_seq_input_grad(const float* dpre, const float* weight, float* dx, int64_t rows, int hidden, int width, void* stream) {
    if (rows < 0 || rows > MAX_GRID || hidden < 1 || hidden > INPUT_HIDDEN || width < 1) return MMN_ERR_ARG;
    if (rows == 0) return MMN_OK;
    if (!dpre || !weight || !dx) return MMN_ERR_ARG;
    const hipStream_t st = (hipStream_t)stream;
    const int64_t ctiles = ceil_div(width, 64), grid = ceil_div(rows, INPUT_ROWS) * ctiles;
    if (grid > MAX_GRID) return MMN_ERR_UNSUPPORTED;
    SEQ_LAUNCH(k_input_grad, dim3((unsigned)grid), dim3(256), 0, st, dpre, weight, dx, rows, hidden, width, (int)ctiles);
    return MMN_OK;
}

}  // extern "C"
