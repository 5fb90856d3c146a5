// Low-rank adapters of many requests beside the shared projections of one network: the forward pass with an
// adapter per row, the gradients of the adapters and their update.  No counterpart in the reference, which has
// one network for everyone; what is shared is its forward and training pass (lib.rs:880-891, 1013-1059).
//
//   h1 = relu(x W1 + b1)                         shared by all rows
//   h2 = tanh(h1 W2 + b2 + u2 B2[s]),  u2 = scale h1 A2[s]
//   l  = h2 W3 + b3 + u3 B3[s],        u3 = scale h2 A3[s]          s = the row's slot
//
//   d3 = p - t            dB3[s] = sum u3^T d3    g3 = scale d3 B3[s]^T    dA3[s] = sum h2^T g3
//   d2 = (d3 W3^T + g3 A3[s]^T)(1 - h2^2)
//                         dB2[s] = sum u2^T d2    g2 = scale d2 B2[s]^T    dA2[s] = sum h1^T g2
//
// The network itself is frozen: no gradient passes below the first adapted projection.
//
// A call's rows are brought into the order of their slots first (a stable counting sort), so that the tiles of
// every product hold rows of one slot, nearly always, and a slot's rows are one range of every row sum.
// Rows are independent of one another in every product: what a row gets does not depend on what the others hold (its place
// in the order may decide which kernel takes it, and with that the order of its sums).
#include <algorithm>
#include <cmath>
#include <new>
#include <type_traits>
#include <vector>

#include "adapt_kernel.h"
#include "adapt_rows.h"
#include "gemm_launch.h"
#include "internal.h"
#include "prof.h"
#include "streamz_hip.h"

namespace sz {

namespace {

using namespace adapt;

// Rows per pass: a call with more is walked in pieces, whose workspace does not grow with it.
constexpr uint64_t kAdaptRows = 131072;

// Calls of up to this many rows go row by row (adapt_rows.h); of half as many in training, whose row kernels do more.
// Forward, on rows and on tiles: 24 and 32 us at 256 rows of 60-512-256-16 with rank 16, 38 and 35 at 512 (rank 32: 38 and 41),
// 52 and 33 at 768; 65 and 90 us at 96 rows of 60-2048-2048-256, 141 and 152 at 512, 201 and 164 at 768.  Training: 56 and
// 72 us at 256 rows of the small network, 73 and 62 at 384; 174 and 194 us of the wide one, 219 and 220.
constexpr uint64_t kFewRows = 512;

inline int round_up(int v, int to) { return (v + to - 1) / to * to; }

bool capturing(hipStream_t s)
{
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    return hipStreamIsCapturing(s, &st) == hipSuccess && st == hipStreamCaptureStatusActive;
}

// Rows per chunk of the factor gradients: enough workgroups (tiles x chunks) to fill the chip twice, no more than 512
// rows (the sums of a chunk's rows are joined by a second launch), no less than 64, or 16 of few rows, whose chunks would hold
// many slots one behind the other (106 rows of 27 slots: 31 us by 16, 41 by 32, 63 by 64; 550 rows of one: 12.4, 10.9, 10.4).
int factor_tiles(const Adapters* a) { return (int)((a->h1 + 63) / 64 + 2 * ((a->h2 + 63) / 64) + (a->out + 63) / 64); }
uint32_t factor_chunk(const Adapters* a, uint64_t rows)
{
    const uint64_t want = std::max<uint64_t>(1, 1024 / factor_tiles(a)), least = rows <= kFewRows ? 16 : 64;
    return (uint32_t)std::min<uint64_t>(512, std::max<uint64_t>(least, (rows / want + least - 1) / least * least));
}
// Most chunks that a call makes whose chunks are shorter than 512 rows: as many as wanted, and those of what is left over by the division of
// the rows among them (fewer rows than chunks are wanted, in chunks of 64 and more).  And that one of up to `rows` rows makes.
uint64_t factor_chunks_any(const Adapters* a)
{
    const uint64_t want = std::max<uint64_t>(1, 1024 / factor_tiles(a));
    return want + want / 64 + 2;
}
uint64_t factor_chunks_most(const Adapters* a, uint64_t rows) { return std::max<uint64_t>((rows + 511) / 512, factor_chunks_any(a)); }

// whether the output layer goes with its rank columns (low_out) instead of being a product of its own
bool low_out_applies(const Adapters* a) { return a->out <= 64; }

// The workspace is in four parts: what a bank needs whatever its calls (the partial gradients of many slots are the largest of
// it), the same for training, and the arrays that go by rows, with those of training by themselves.  Only the latter two grow.
enum Part { PART_BANK, PART_TRAIN_BANK, PART_ROWS, PART_TRAIN_ROWS };

// How the arrays of a part for `rows` rows lie; `base` null: only the size.
size_t lay_out(const Adapters* a, Part part, uint64_t rows, char* base, AdaptWorkspace& o)
{
    size_t at = 0;
    auto take = [&](auto*& p, uint64_t count) {
        p = reinterpret_cast<std::decay_t<decltype(p)>>(base + at);
        at += (count * sizeof(*p) + 255) / 256 * 256;
    };
    const uint64_t blocks = (rows + kGroupRows - 1) / kGroupRows, S = a->slots;
    o.ldx = round_up((int)a->in, 32);
    o.ld1 = round_up((int)a->h1, 32); o.ld2 = round_up((int)a->h2, 32); o.ld3 = round_up((int)std::max(a->out, 1u), 4);
    o.ldu = round_up((int)a->rank, 8);
    switch (part) {
    case PART_BANK:
        take(o.begin, S + 2); take(o.total, S + 1);
        take(o.add2, kFewRows * o.ld2); take(o.add3, kFewRows * o.ld3);
        take(o.w2t, (uint64_t)o.ld1 * a->h2);
        if (!low_out_applies(a)) take(o.w3t, (uint64_t)o.ld2 * a->out);
        take(o.w2s, 3 * ((uint64_t)a->h1 * a->h2 + 1) / 2 + 4);
        break;
    case PART_TRAIN_BANK:
        take(o.slot_slab, S * a->per_slot());
        o.chunks = factor_chunks_any(a);
        take(o.chunk_slab, o.chunks * a->per_slot());
        break;
    case PART_ROWS:
        take(o.order, rows); take(o.row_slot, rows); take(o.count, (S + 1) * blocks);
        take(o.xs, rows * o.ldx); take(o.live0, rows);
        take(o.h1, (rows + 32) * o.ld1); take(o.h2, (rows + 32) * o.ld2); take(o.lg, (rows + 32) * o.ld3);
        take(o.u2, rows * o.ldu); take(o.u3, rows * o.ldu);
        break;
    default:
        take(o.live, rows); take(o.loss, rows);
        take(o.d2, (rows + 32) * o.ld2); take(o.g2, rows * o.ldu); take(o.g3, rows * o.ldu);
        if (factor_chunks_most(a, rows) > factor_chunks_any(a)) {  // (else those of the bank are enough)
            o.chunks = factor_chunks_most(a, rows);
            take(o.chunk_slab, o.chunks * a->per_slot());
        }
    }
    return at;
}

// Arrays that grow are at least doubled, and beyond half of the most rows become the largest at once: the earlier ones, which stay,
// are together no larger than the last.
uint64_t grown(uint64_t rows, uint64_t have)
{
    rows = std::max<uint64_t>((rows + 255) / 256 * 256, 256);
    if (have) rows = std::max<uint64_t>(rows, 2 * have);
    return rows > kAdaptRows || (have && rows > kAdaptRows / 2) ? kAdaptRows : rows;
}

int ensure(Adapters* a, uint64_t rows, bool training, hipStream_t s)
{
    rows = std::min<uint64_t>(std::max<uint64_t>(rows, 1), kAdaptRows);
    const Part parts[] = {PART_BANK, PART_TRAIN_BANK, PART_ROWS, PART_TRAIN_ROWS};
    const uint64_t need[] = {1, training ? 1u : 0u, rows, training ? rows : 0};
    AdaptWorkspace w = a->ws;
    uint64_t get[4] = {};
    size_t bytes = 0;
    for (const Part p : parts) {
        if (a->ws_have[p] >= need[p]) continue;
        get[p] = p == PART_ROWS || p == PART_TRAIN_ROWS ? grown(need[p], a->ws_have[p]) : 1;
        bytes += lay_out(a, p, get[p], nullptr, w);
    }
    if (bytes == 0) return SZH_OK;
    if (capturing(s)) { set_error("adapters: the workspace must be reserved before a stream is captured (szh_adapters_reserve)"); return SZH_EINVAL; }
    char* at = nullptr;
    SZ_HIP(hipMalloc((void**)&at, bytes));
    try { a->arenas.push_back(at); } catch (...) { (void)hipFree(at); throw; }
    SZ_HIP(hipMemset(at, 0, bytes));  // the columns between a row's end and its stride are read as zeros
    SZ_HIP(hipDeviceSynchronize());
    // the old arrays stay until the handle goes: a captured graph may still work in them
    for (const Part p : parts) {
        if (!get[p]) continue;
        at += lay_out(a, p, get[p], at, a->ws);
        a->ws_have[p] = get[p];
    }
    return SZH_OK;
}

int check_pair(const Net* n, const Adapters* a)
{
    if (n->in != a->in || n->h1 != a->h1 || n->h2 != a->h2 || n->out != a->out) {
        set_error("adapters were made for a network %u-%u-%u-%u, this one is %u-%u-%u-%u", a->in, a->h1, a->h2, a->out, n->in, n->h1,
                  n->h2, n->out);
        return SZH_EINVAL;
    }
    if (n->device != a->device) { set_error("adapters and network are on different devices"); return SZH_EINVAL; }
    return SZH_OK;
}

bool overlap(const float* a, uint64_t a_len, const float* b, uint64_t b_len) { return a < b + b_len && b < a + a_len; }

int group_rows(Adapters* a, const int32_t* slots_dev, uint32_t rows, hipStream_t s)
{
    AdaptWorkspace& w = a->ws;
    const int S = (int)a->slots, blocks = (int)((rows + kGroupRows - 1) / kGroupRows);
    const size_t lds = (S + 1) * sizeof(uint32_t);
    ProfScope prof("adapt_group", s);
    if (blocks == 1) {
        hipLaunchKernelGGL(group_few_kernel, dim3(1), dim3(64), lds, s, slots_dev, rows, S, w.begin, w.order, w.row_slot);
        SZ_HIP(hipGetLastError());
        return SZH_OK;
    }
    if (blocks <= kGroupWaves && S <= kGroupMidSlots) {
        const size_t mid = (size_t)kGroupWaves * (S + 1) * sizeof(uint32_t);
        if (int rc = allow_dynamic_lds((const void*)group_mid_kernel, mid)) return rc;
        hipLaunchKernelGGL(group_mid_kernel, dim3(1), dim3(64 * kGroupWaves), mid, s, slots_dev, rows, S, w.begin, w.order, w.row_slot);
        SZ_HIP(hipGetLastError());
        return SZH_OK;
    }
    hipLaunchKernelGGL(group_count_kernel, dim3(blocks), dim3(64), lds, s, slots_dev, rows, S, blocks, w.count);
    hipLaunchKernelGGL(group_scan_kernel, dim3(S + 1), dim3(64), 0, s, w.count, blocks, w.total);
    hipLaunchKernelGGL(group_begin_kernel, dim3(1), dim3(64), 0, s, w.total, S, rows, w.begin);
    hipLaunchKernelGGL(group_place_kernel, dim3(blocks), dim3(64), lds, s, slots_dev, rows, S, blocks, w.count, w.begin, w.order, w.row_slot);
    SZ_HIP(hipGetLastError());
    return SZH_OK;
}

// whether rows of `width` values, `apart` values from one to the next, can be read in aligned pieces of 16 bytes
bool in_fours(const float* p, uint64_t width, uint64_t apart) { return width % 4 == 0 && apart % 4 == 0 && ((uintptr_t)p & 15) == 0; }

template <int NT, int OT, int WAVES, int UNR, bool FOURS = false>
int launch_low(LowArgs g, hipStream_t s)
{
    constexpr size_t lds = (size_t)WAVES * 32 * NT * 16 * sizeof(float);
    if (int rc = allow_dynamic_lds((const void*)low_kernel<NT, OT, WAVES, UNR, FOURS>, lds)) return rc;
    const unsigned tiles = (g.rows + 31) / 32;
    g.parts = tiles >= 512 ? 1 : (int)std::min<unsigned>(32, 1024 / tiles);
    hipLaunchKernelGGL((low_kernel<NT, OT, WAVES, UNR, FOURS>), dim3(tiles, g.parts), dim3(64 * WAVES), lds, s, g);
    SZ_HIP(hipGetLastError());
    return SZH_OK;
}

// u = scale * x F[slot]
int low_product(const Adapters* a, const float* x, int ldx, int K, const float* factor, int f_k, int f_j, uint32_t rows, float* u,
                hipStream_t s)
{
    LowArgs g{};
    g.x = x; g.ldx = ldx; g.K = K; g.factor = factor; g.factor_slot = a->per_slot(); g.f_k = f_k; g.f_j = f_j;
    g.rank = (int)a->rank; g.row_slot = a->ws.row_slot; g.rows = rows; g.u = u; g.ldu = a->ws.ldu; g.scale = a->scale;
    ProfScope prof("adapt_low", s);
    const bool fours = f_k == 1 && in_fours(factor, f_j, g.factor_slot);
    switch ((a->rank + 15) / 16 * 2 + fours) {
    case 2: return launch_low<1, 0, 4, 4>(g, s);
    case 3: return launch_low<1, 0, 4, 4, true>(g, s);
    case 4: return launch_low<2, 0, 4, 2>(g, s);
    case 5: return launch_low<2, 0, 8, 4, true>(g, s);
    case 6: return launch_low<3, 0, 4, 2>(g, s);
    case 7: return launch_low<3, 0, 4, 2, true>(g, s);
    case 8: return launch_low<4, 0, 4, 2>(g, s);
    default: return launch_low<4, 0, 4, 2, true>(g, s);
    }
}

// h1 and u2 in one pass over x, straight from the caller's rows where `order` is given.  At rank 32 a wave's W1 and A2 leave
// no registers for the rows to come, and the pass takes as long as the gather and the two products it replaces.
bool front_applies(const Net* n, const Adapters* a) { return n->in <= kFrontIn && n->h1 <= 64 * kFrontWaves && a->rank <= 16; }
int front_rows(const Net* n, const Adapters* a, const float* x, int ldx, const uint32_t* order, uint8_t* live, uint32_t rows, hipStream_t s)
{
    const AdaptWorkspace& w = a->ws;
    FrontArgs g{};
    g.x = x; g.order = order; g.w1 = n->d_params + n->off_w1(); g.b1 = n->d_params + n->off_b1(); g.a2 = a->d_params + a->off_a2();
    g.per_slot = a->per_slot(); g.row_slot = w.row_slot; g.h1 = w.h1; g.u2 = w.u2; g.live = live; g.rows = rows;
    g.in = (int)n->in; g.ldx = ldx; g.n1 = (int)n->h1; g.ld1 = w.ld1; g.rank = (int)a->rank; g.ldu = w.ldu; g.scale = a->scale;
    const bool fours = in_fours(x, n->in, ldx) && in_fours(g.w1, n->h1, n->h1) && in_fours(g.b1, n->h1, 0);
    const int waves = (g.n1 + 63) / 64;
    const size_t lds = (size_t)2 * kFrontGroup * waves * 16 * 17 * sizeof(float);
    if (int rc = allow_dynamic_lds(fours ? (const void*)front_kernel<true> : (const void*)front_kernel<false>, lds)) return rc;
    const dim3 grid(std::min<unsigned>((rows + 15) / 16, (unsigned)compute_units() * (kFrontWaves / waves))), block(64 * waves);
    ProfScope prof("adapt_h1", s);
    if (fours) hipLaunchKernelGGL((front_kernel<true>), grid, block, lds, s, g);
    else hipLaunchKernelGGL((front_kernel<false>), grid, block, lds, s, g);
    SZ_HIP(hipGetLastError());
    return SZH_OK;
}

// u3 and the logits of up to 64 classes in one pass over h2
int low_out(const Net* n, const Adapters* a, uint32_t rows, hipStream_t s)
{
    const AdaptWorkspace& w = a->ws;
    LowArgs g{};
    g.x = w.h2; g.ldx = w.ld2; g.K = (int)n->h2; g.factor = a->d_params + a->off_a3(); g.factor_slot = a->per_slot();
    g.f_k = (int)a->rank; g.f_j = 1; g.rank = (int)a->rank; g.row_slot = w.row_slot; g.rows = rows; g.u = w.u3; g.ldu = w.ldu; g.scale = a->scale;
    g.W = n->d_params + n->off_w3(); g.bias = n->d_params + n->off_b3(); g.up = a->d_params + a->off_b3(); g.up_slot = a->per_slot();
    g.y = w.lg; g.out = (int)n->out; g.ldy = w.ld3;
    ProfScope prof("adapt_out", s);
    const int rt = (int)(a->rank + 15) / 16, ot = (int)(n->out + 15) / 16;
    // (three tiles are taken as four: a column tile without columns repeats the last one's)
    switch ((ot > 2 ? 4 : ot) * 8 + (rt > 2 ? 4 : rt)) {
    case 1 * 8 + 1: return launch_low<2, 1, 4, 2>(g, s);
    case 1 * 8 + 2: return launch_low<3, 1, 8, 2>(g, s);
    case 1 * 8 + 4: return launch_low<5, 1, 4, 1>(g, s);
    case 2 * 8 + 1: return launch_low<3, 2, 8, 2>(g, s);
    case 2 * 8 + 2: return launch_low<4, 2, 4, 2>(g, s);
    case 2 * 8 + 4: return launch_low<6, 2, 4, 1>(g, s);
    case 4 * 8 + 1: return launch_low<5, 4, 4, 1>(g, s);
    case 4 * 8 + 2: return launch_low<6, 4, 4, 1>(g, s);
    default: return launch_low<8, 4, 4, 1>(g, s);
    }
}

// the gradients of a pass's four factors, its losses and live rows, added to the bank's
int factor_gradients(Adapters* a, uint32_t rows, hipStream_t s)
{
    const AdaptWorkspace& w = a->ws;
    const int h1 = (int)a->h1, h2 = (int)a->h2, out = (int)a->out, r = (int)a->rank;
    FactorArgs g{};
    g.ldw = w.ldu; g.rank = r; g.slots = (int)a->slots; g.begin = w.begin; g.row_slot = w.row_slot; g.live = w.live;
    g.job[0] = {w.h1, w.g2, nullptr, nullptr, a->off_a2(), w.ld1, h1, r, 1, 0, 0};
    g.job[1] = {w.d2, w.u2, nullptr, nullptr, a->off_b2(), w.ld2, h2, 1, h2, 0, 0};
    g.job[2] = {w.h2, w.g3, nullptr, nullptr, a->off_a3(), w.ld2, h2, r, 1, 0, 0};
    g.job[3] = {w.lg, w.u3, nullptr, nullptr, a->off_b3(), w.ld3, out, 1, out, 0, 0};
    g.chunk = factor_chunk(a, rows);
    const uint64_t chunks = (rows + g.chunk - 1) / g.chunk;
    if (chunks > w.chunks) { set_error("adapters: more chunks than the workspace holds"); return SZH_EINVAL; }
    float *slot_slab = w.slot_slab, *chunk_slab = w.chunk_slab;
    int tiles = 0, blocks = 0;
    for (FactorJob& j : g.job) {
        j.first = tiles; j.first_out = blocks; j.slot_slab = slot_slab; j.chunk_slab = chunk_slab;
        tiles += (j.M + 63) / 64;
        blocks += (j.M * r + 255) / 256;
        slot_slab += a->slots * (uint64_t)j.M * r;
        chunk_slab += chunks * (uint64_t)j.M * r;
    }
    const dim3 grid(tiles, (unsigned)chunks), block(256);
    ProfScope prof("adapt_grad", s);
    switch ((r + 15) / 16) {
    case 1: hipLaunchKernelGGL((factor_grad_kernel<1, 4>), grid, block, 0, s, g); break;
    case 2: hipLaunchKernelGGL((factor_grad_kernel<2, 4>), grid, block, 0, s, g); break;
    case 3: hipLaunchKernelGGL((factor_grad_kernel<3, 2>), grid, block, 0, s, g); break;
    default: hipLaunchKernelGGL((factor_grad_kernel<4, 2>), grid, block, 0, s, g); break;
    }
    hipLaunchKernelGGL(factor_reduce_kernel, dim3(blocks + 1, a->slots), block, 0, s, g, a->d_grad, a->per_slot(), w.loss, w.live, a->d_sums,
                       a->d_grad + a->per_slot() * a->slots);
    SZ_HIP(hipGetLastError());
    return SZH_OK;
}

BackArgs back_args(const Net* n, const Adapters* a, uint32_t rows)
{
    const AdaptWorkspace& w = a->ws;
    const float* F = a->d_params;
    BackArgs g{};
    g.d3 = w.lg; g.h2 = w.h2; g.w3 = n->d_params + n->off_w3(); g.a3 = F + a->off_a3(); g.b3 = F + a->off_b3(); g.b2 = F + a->off_b2();
    g.per_slot = a->per_slot(); g.row_slot = w.row_slot; g.d2 = w.d2; g.g2 = w.g2; g.g3 = w.g3; g.rows = rows;
    g.n2 = (int)n->h2; g.out = (int)n->out; g.rank = (int)a->rank; g.ld2 = w.ld2; g.ld3 = w.ld3; g.ldu = w.ldu; g.scale = a->scale;
    return g;
}
bool back_fours(const Adapters* a, const BackArgs& g)
{
    return in_fours(g.w3, g.out, g.out) && in_fours(g.a3, a->rank, g.per_slot) && in_fours(g.b2, g.n2, g.per_slot);
}

// The output layer, the loss and back to d2 and the rank columns in one launch, lg taking d3
bool tail_applies(const Adapters* a) { return a->out <= 64 && a->rank <= 16; }
template <int OT, int WAVES, int T>
int launch_tail(const BackArgs& g, bool fours, const TailArgs& o, const Controls& ctl, const ControlRun& c, hipStream_t s)
{
    const dim3 grid((g.rows + 16 * T - 1) / (16 * T)), block(64 * WAVES);
    ProfScope prof("adapt_tail", s);
    if (fours) hipLaunchKernelGGL((tail_kernel<OT, WAVES, T, true>), grid, block, 0, s, g, o, ctl, c);
    else hipLaunchKernelGGL((tail_kernel<OT, WAVES, T, false>), grid, block, 0, s, g, o, ctl, c);
    SZ_HIP(hipGetLastError());
    return SZH_OK;
}
int tail_rows(const Net* n, const Adapters* a, const Controls& ctl, const ControlRun& c, uint32_t rows, hipStream_t s)
{
    const BackArgs g = back_args(n, a, rows);
    const TailArgs o{n->d_params + n->off_b3(), a->ws.u3, a->ws.lg};
    const bool fours = back_fours(a, g);
    // (as long as a compute unit has at most one workgroup: fewer rows and more waves for them.  1056 rows x 2048 units 49 us, 68 on
    // 32 rows and eight waves; 550 x 256 12.8, 13.6, and 17 on four waves)
    const unsigned cus = (unsigned)compute_units();
    if (rows <= 16 * cus) {
        if (n->out <= 16) return launch_tail<1, 16, 1>(g, fours, o, ctl, c, s);
        if (n->out <= 32) return launch_tail<2, 16, 1>(g, fours, o, ctl, c, s);
        return launch_tail<4, 8, 1>(g, fours, o, ctl, c, s);
    }
    if (n->out <= 16) return rows <= 32 * cus ? launch_tail<1, 8, 2>(g, fours, o, ctl, c, s) : launch_tail<1, 4, 2>(g, fours, o, ctl, c, s);
    if (n->out <= 32) return rows <= 32 * cus ? launch_tail<2, 8, 2>(g, fours, o, ctl, c, s) : launch_tail<2, 4, 2>(g, fours, o, ctl, c, s);
    return launch_tail<4, 4, 2>(g, fours, o, ctl, c, s);
}

// d3 -> g3, d2, g2 in one launch; up to 64 classes (beyond them the product with w3 wants larger tiles)
bool back_applies(const Adapters* a) { return a->out <= 64; }
int back_rows(const Net* n, const Adapters* a, uint32_t rows, hipStream_t s)
{
    const BackArgs g = back_args(n, a, rows);
    const bool fours = back_fours(a, g);
    ProfScope prof("adapt_back", s);
    if (rows <= 16u * (unsigned)compute_units()) {  // (fewer tiles than compute units: half the rows, and eight waves for them)
        const dim3 grid((rows + 15) / 16), block(512);
        switch ((a->rank + 15) / 16 * 2 + fours) {
        case 2: hipLaunchKernelGGL((back_kernel<1, 8, 1, false>), grid, block, 0, s, g); break;
        case 3: hipLaunchKernelGGL((back_kernel<1, 8, 1, true>), grid, block, 0, s, g); break;
        case 4: hipLaunchKernelGGL((back_kernel<2, 8, 1, false>), grid, block, 0, s, g); break;
        case 5: hipLaunchKernelGGL((back_kernel<2, 8, 1, true>), grid, block, 0, s, g); break;
        case 6: hipLaunchKernelGGL((back_kernel<3, 8, 1, false>), grid, block, 0, s, g); break;
        case 7: hipLaunchKernelGGL((back_kernel<3, 8, 1, true>), grid, block, 0, s, g); break;
        case 8: hipLaunchKernelGGL((back_kernel<4, 8, 1, false>), grid, block, 0, s, g); break;
        default: hipLaunchKernelGGL((back_kernel<4, 8, 1, true>), grid, block, 0, s, g); break;
        }
        SZ_HIP(hipGetLastError());
        return SZH_OK;
    }
    const dim3 grid((rows + 31) / 32);
    switch ((a->rank + 15) / 16 * 2 + fours) {
    case 2: hipLaunchKernelGGL((back_kernel<1, 4, 2, false>), grid, dim3(256), 0, s, g); break;
    case 3: hipLaunchKernelGGL((back_kernel<1, 4, 2, true>), grid, dim3(256), 0, s, g); break;
    case 4: hipLaunchKernelGGL((back_kernel<2, 8, 2, false>), grid, dim3(512), 0, s, g); break;
    case 5: hipLaunchKernelGGL((back_kernel<2, 8, 2, true>), grid, dim3(512), 0, s, g); break;
    case 6: hipLaunchKernelGGL((back_kernel<3, 4, 2, false>), grid, dim3(256), 0, s, g); break;
    case 7: hipLaunchKernelGGL((back_kernel<3, 4, 2, true>), grid, dim3(256), 0, s, g); break;
    case 8: hipLaunchKernelGGL((back_kernel<4, 4, 2, false>), grid, dim3(256), 0, s, g); break;
    default: hipLaunchKernelGGL((back_kernel<4, 4, 2, true>), grid, dim3(256), 0, s, g); break;
    }
    SZ_HIP(hipGetLastError());
    return SZH_OK;
}

void adapt_args(GemmArgs& g, const Adapters* a, const float* low, const float* up, int up_k, int up_n)
{
    g.low = low; g.ld_low = a->ws.ldu; g.up = up; g.up_slot = a->per_slot(); g.up_k = up_k; g.up_n = up_n; g.rank = (int)a->rank;
    g.row_slot = a->ws.row_slot; g.row_begin = a->ws.begin;
}

template <bool TANH>
int thin_product(const float* A, int lda, int K, const float* W, const float* add, int ldadd, const float* bias, float* C, int ldc, int N,
                 uint32_t rows, const char* tag, hipStream_t s)
{
    ThinArgs g{};
    g.A = A; g.lda = lda; g.W = W; g.add = add; g.ldadd = ldadd; g.bias = bias; g.C = C; g.ldc = ldc; g.M = (int)rows; g.N = N; g.K = K;
    ProfScope prof(tag, s);
    hipLaunchKernelGGL((thin_kernel<TANH>), dim3((N + 31) / 32, (rows + 31) / 32), dim3(64 * kThinWaves), 0, s, g);
    SZ_HIP(hipGetLastError());
    return SZH_OK;
}

// Which kernels a shared product of `rows` rows goes to.  The 256 x 256 tiles of gemm_f32w_kernel are the fastest
// (137 TFLOP/s) but run one per compute unit, so only whole rounds of them pay: the first rows go there, the rest to
// what is quickest for so many.  Times in us of a product [rows][K] x [K][N], fitted to measurements over K 512 .. 2048,
// N 256 .. 2048, 256 to 66140 rows (66140 x 512 x 256: 182 us on 64-row tiles, 283 on 256-row tiles, 145 split;
// 26456 x 2048 x 2048: 1849, 2051, 1660):
//   256-row tiles: 0.232 K + 18 for every round of one tile per compute unit
//   128-row tiles: two per unit 0.122 K + 17, one 0.071 K + 12        64-row tiles: 0.0337 K + 4 each, once 0.0085 K
//   32 x 32 thin tiles: 5 + 0.001 K, and 3.55e-5 K each
// These are of the product alone: the rank columns added behind it are in no term.  With rank 16 the 145 us above are 180 (172 and 8); at
// 13228 x 2048 x 2048 with rank 32 the round of 256-row tiles takes 587 instead of 499, the 64-row tiles beside it 416 instead of 382.
struct ProductPart { int how; uint32_t rows; };   // how: 256, 128 or 64 rows a tile, 0 thin
struct ProductPlan { ProductPart part[3]; int parts; double time; };

double part_time(int how, uint32_t rows, int N, int K, double cus)
{
    auto ceil_div = [](uint64_t a, uint64_t b) { return (double)((a + b - 1) / b); };
    if (how == 0) return 5 + 0.001 * K + ceil_div(rows, 32) * ceil_div(N, 32) * 3.55e-5 * K;
    if (how == 256) return std::ceil(ceil_div(rows, 256) * ceil_div(N, 256) / cus) * (0.232 * K + 18) + 6;  // (W transposed first: a launch)
    const double c = std::ceil(ceil_div(rows, how) * ceil_div(N, 128) / cus);
    if (how == 64) return c * (0.0337 * K + 4) + 0.0085 * K;
    return std::floor(c / 2) * (0.122 * K + 17) + (std::fmod(c, 2.0) != 0 ? 0.071 * K + 12 : 0);
}
// The quickest of: one kernel for all rows, or whole rounds of tiles of `most` rows or fewer first and the rest the same way
// (1056 x 2048 x 2048: 178 us on 64-row tiles alone, whose second round is one row of tiles, 115 with that left to thin ones).
ProductPlan plan_rows(uint32_t rows, int N, int K, double cus, int most)
{
    ProductPlan best{{{0, rows}}, 1, part_time(0, rows, N, K, cus)};
    for (const int how : {64, 128, 256}) {
        if (how > most) continue;
        const double all = part_time(how, rows, N, K, cus);
        if (all < best.time) best = {{{how, rows}}, 1, all};
        const uint64_t across = ((uint64_t)N + (how == 256 ? 255 : 127)) / (how == 256 ? 256 : 128), down = ((uint64_t)rows + how - 1) / how;
        const uint64_t first = (uint64_t)(across * down / (uint64_t)cus) * (uint64_t)cus / across * how;  // rows of the whole rounds
        if (first == 0 || first >= rows) continue;
        const ProductPlan rest = plan_rows(rows - (uint32_t)first, N, K, cus, how == 256 ? 128 : 0);
        const double time = part_time(how, (uint32_t)first, N, K, cus) + rest.time + 2;
        if (time >= best.time) continue;
        best = {{{how, (uint32_t)first}}, 1 + rest.parts, time};
        for (int i = 0; i < rest.parts; ++i) best.part[1 + i] = rest.part[i];
    }
    return best;
}

// C = epilogue(A W + low part), rows sorted by slot, as planned.  g: the whole product with B = W [K][N]; Kp: A's
// columns with the zeros behind them, a multiple of 32; wt: room for W transposed and padded, [N][Kp].
template <int EPI, int TAG>
int shared_product(const GemmArgs& g, int Kp, float* wt, hipStream_t s)
{
    const ProductPlan p = plan_rows((uint32_t)g.M, g.N, g.K, compute_units(), 256);
    GemmArgs h = g;
    for (int i = 0; i < p.parts; ++i) {
        h.M = (int)p.part[i].rows;
        int rc = SZH_OK;
        if (p.part[i].how == 256) {
            {
                ProfScope prof("w2t", s);
                hipLaunchKernelGGL(pad_transpose_kernel, dim3((unsigned)(((uint64_t)g.N * Kp + 255) / 256)), dim3(256), 0, s, g.B, g.K, g.N, Kp, wt);
                SZ_HIP(hipGetLastError());
            }
            GemmArgs w = h;
            w.B = wt; w.ldb = Kp; w.K = w.k_chunk = Kp;
            rc = launch_gemm_f32w<EPI, TAG>(w, s);
        } else if (p.part[i].how == 64) {
            rc = launch_gemm_rows<A_ROWS, B_KROWS, EPI, TAG, 64>(h, s);
        } else if (p.part[i].how == 128) {
            rc = launch_gemm_rows<A_ROWS, B_KROWS, EPI, TAG, 128>(h, s);
        } else {
            ThinArgs t{};
            t.A = h.A; t.lda = h.lda; t.W = h.B; t.bias = h.bias; t.C = h.C; t.ldc = h.ldc; t.M = h.M; t.N = h.N; t.K = h.K;
            t.low = h.low; t.up = h.up; t.row_slot = h.row_slot; t.up_slot = h.up_slot; t.ld_low = h.ld_low; t.rank = h.rank;
            ProfScope prof(kGemmTagName[TAG], s);
            hipLaunchKernelGGL((thin_kernel<EPI == EPI_ADAPT_TANH>), dim3((t.N + 31) / 32, (t.M + 31) / 32), dim3(64 * kThinWaves), 0, s, t);
            SZ_HIP(hipGetLastError());
        }
        if (rc) return rc;
        const uint32_t m = p.part[i].rows;
        h.A += (size_t)m * g.lda; h.C += (size_t)m * g.ldc; h.low += (size_t)m * g.ld_low; h.row_slot += m;
    }
    return SZH_OK;
}

// logits of `rows` grouped rows in the workspace's lg, activations in h1, h2, rank columns in u2, u3; x, in the caller's
// order, unless gather_rows has put its rows into xs already (null); `tail`: as far as h2
int forward_rows(Net* n, Adapters* a, const float* x, uint8_t* live, bool tail, uint32_t rows, hipStream_t s)
{
    AdaptWorkspace& w = a->ws;
    const float* P = n->d_params;
    const float* F = a->d_params;
    const int r = (int)a->rank;
    int rc;
    GemmArgs g{};
    if (front_applies(n, a)) {
        rc = x ? front_rows(n, a, x, (int)n->in, w.order, live, rows, s) : front_rows(n, a, w.xs, w.ldx, nullptr, nullptr, rows, s);
    } else {
        g.A = w.xs; g.lda = w.ldx; g.C = w.h1; g.ldc = w.ld1; g.M = (int)rows; g.N = (int)n->h1; g.bias = P + n->off_b1();
        g.B = P + n->off_w1(); g.ldb = (int)n->h1; g.K = g.k_chunk = (int)n->in;
        // (a short k: 64-row tiles are never behind, 57 us against 61 on 128 and 70 on 256 rows at 66140 x 60 x 512)
        rc = launch_gemm_rows<A_ROWS, B_KROWS, EPI_BIAS_RELU, T_ADAPT1, 64>(g, s);
        if (!rc) rc = low_product(a, w.h1, w.ld1, (int)n->h1, F + a->off_a2(), r, 1, rows, w.u2, s);
    }
    if (rc) return rc;
    g = GemmArgs{};
    g.A = w.h1; g.lda = w.ld1; g.C = w.h2; g.ldc = w.ld2; g.M = (int)rows; g.N = (int)n->h2; g.K = g.k_chunk = (int)n->h1;
    g.B = P + n->off_w2(); g.ldb = (int)n->h2; g.bias = P + n->off_b2();
    adapt_args(g, a, w.u2, F + a->off_b2(), (int)n->h2, 1);
    if (use_x3(n, rows)) {
        {
            ProfScope prof("w2split", s);
            const uint64_t count = (uint64_t)n->h1 * n->h2;
            hipLaunchKernelGGL(transpose_kernel, dim3((n->h2 + 31) / 32, (n->h1 + 31) / 32), dim3(256), 0, s, P + n->off_w2(), (int)n->h1,
                               (int)n->h2, w.w2t);
            hipLaunchKernelGGL(split_planes_kernel, dim3((unsigned)((count / 2 + 255) / 256)), dim3(256), 0, s, w.w2t, count, w.w2s, count / 2);
            SZ_HIP(hipGetLastError());
        }
        g.B = (const float*)w.w2s; g.ldb = (int)n->h1; g.b_plane = (uint64_t)n->h1 * n->h2;
        rc = launch_gemm_x3<X3_ROWS_F32, X3_ROWS_SPLIT, EPI_ADAPT_TANH, T_ADAPT2>(g, 1, s);
    } else {
        rc = shared_product<EPI_ADAPT_TANH, T_ADAPT2>(g, w.ld1, w.w2t, s);
    }
    if (rc || n->out == 0 || tail) return rc;
    if (low_out_applies(a)) return low_out(n, a, rows, s);
    rc = low_product(a, w.h2, w.ld2, (int)n->h2, F + a->off_a3(), r, 1, rows, w.u3, s);
    if (rc) return rc;
    g = GemmArgs{};
    g.A = w.h2; g.lda = w.ld2; g.C = w.lg; g.ldc = w.ld3; g.M = (int)rows; g.N = (int)n->out; g.K = g.k_chunk = (int)n->h2;
    g.B = P + n->off_w3(); g.ldb = (int)n->out; g.bias = P + n->off_b3();
    adapt_args(g, a, w.u3, F + a->off_b3(), (int)n->out, 1);
    return shared_product<EPI_ADAPT_BIAS, T_ADAPT3>(g, w.ld2, w.w3t, s);
}

// Whether a call takes the few-row path: its row kernels hold a row's activations in LDS.
bool few_rows(const Net* n, uint64_t rows, bool training)
{
    return rows <= (training ? kFewRows / 2 : kFewRows) && n->in + n->h1 + 2 * n->h2 + n->out <= 24576;
}

// w3 beyond this is not streamed by every row: the logits become a product of their own
constexpr uint64_t kRowOutFloats = 65536;

RowArgs row_args(const Net* n, Adapters* a, const float* x, uint64_t ldx, const int32_t* slot)
{
    const AdaptWorkspace& w = a->ws;
    const float* P = n->d_params;
    RowArgs g{};
    g.x = x; g.ldx = ldx; g.w1 = P + n->off_w1(); g.b1 = P + n->off_b1(); g.w3 = P + n->off_w3(); g.b3 = P + n->off_b3();
    g.factors = a->d_params; g.per_slot = a->per_slot();
    g.off_a2 = a->off_a2(); g.off_b2 = a->off_b2(); g.off_a3 = a->off_a3(); g.off_b3 = a->off_b3();
    g.slot = slot; g.slots = (int)a->slots; g.in = (int)n->in; g.n1 = (int)n->h1; g.n2 = (int)n->h2; g.out = (int)n->out;
    g.rank = (int)a->rank; g.ldu = w.ldu; g.ld1 = w.ld1; g.ld2 = w.ld2; g.ld3 = w.ld3; g.scale = a->scale;
    g.h1 = w.h1; g.h2 = w.h2; g.add2 = w.add2; g.add3 = w.add3;
    return g;
}

template <int OUT>
int launch_row_out(const RowArgs& g, const Controls& ctl, const ControlRun& c, uint32_t rows, hipStream_t s)
{
    const size_t lds = (kRowPart + 2 * g.n2 + 64 + g.out) * sizeof(float);
    if (int rc = allow_dynamic_lds((const void*)row_out_kernel<OUT>, lds)) return rc;
    ProfScope prof("adapt_row_out", s);
    hipLaunchKernelGGL((row_out_kernel<OUT>), dim3(rows), dim3(kRowT), lds, s, g, ctl, c);
    SZ_HIP(hipGetLastError());
    return SZH_OK;
}

// The call of few rows, in the caller's order; c holds what it wants of the logits (by row).
int forward_few(Net* n, Adapters* a, const float* x, uint64_t ldx, const int32_t* slot, uint32_t rows, const Controls& ctl, const ControlRun& c,
                float* u2, float* u3, hipStream_t s)
{
    AdaptWorkspace& w = a->ws;
    const float* P = n->d_params;
    RowArgs g = row_args(n, a, x, ldx, slot);
    g.u2 = u2; g.u3 = u3;
    const size_t lds = (kRowPart + g.n1 + 64 + g.in) * sizeof(float);
    if (int rc = allow_dynamic_lds((const void*)row_hidden_kernel, lds)) return rc;
    {
        ProfScope prof("adapt_row_h1", s);
        hipLaunchKernelGGL(row_hidden_kernel, dim3(rows), dim3(kRowT), lds, s, g);
        SZ_HIP(hipGetLastError());
    }
    int rc = thin_product<true>(w.h1, w.ld1, (int)n->h1, P + n->off_w2(), w.add2, w.ld2, P + n->off_b2(), w.h2, w.ld2, (int)n->h2, rows,
                                "adapt_h2", s);
    if (rc) return rc;
    const bool train = c.labels != nullptr;
    if ((uint64_t)n->h2 * n->out <= kRowOutFloats) {
        if (train) { g.g2 = w.g2; g.g3 = w.g3; g.d2 = w.d2; g.d3 = w.lg; return launch_row_out<OUT_TRAIN>(g, ctl, c, rows, s); }
        return launch_row_out<OUT_INFER>(g, ctl, c, rows, s);
    }
    rc = launch_row_out<OUT_ADD>(g, ctl, c, rows, s);
    if (!rc) rc = thin_product<false>(w.h2, w.ld2, (int)n->h2, P + n->off_w3(), w.add3, w.ld3, P + n->off_b3(), w.lg, w.ld3, (int)n->out, rows,
                                      "adapt_out", s);
    return rc ? rc : control_run(ctl, c, s);
}

int gather_rows(Adapters* a, const float* x, uint32_t rows, float dropout, uint64_t seed, uint64_t counter0, uint8_t* live, hipStream_t s)
{
    ProfScope prof("prep", s);
    hipLaunchKernelGGL(gather_rows_kernel, dim3((rows + 3) / 4), dim3(256), 0, s, x, a->ws.order, rows, (int)a->in, dropout, seed, counter0,
                       a->ws.xs, a->ws.ldx, live);
    SZ_HIP(hipGetLastError());
    return SZH_OK;
}

// the controls of the call's rows from row r0 on
Controls from_row(const Controls& c, uint64_t r0)
{
    Controls d = c;
    if (d.set_of_row) d.set_of_row += r0;
    return d;
}

// one pass of a forward or vote call
int infer_rows(Net* n, Adapters* a, const float* x, const int32_t* slots_dev, uint32_t rows, const Controls& ctl, ControlRun c, hipStream_t s)
{
    if (few_rows(n, rows, false)) return forward_few(n, a, x, n->in, slots_dev, rows, ctl, c, nullptr, nullptr, s);
    int rc = group_rows(a, slots_dev, rows, s);
    const bool front = front_applies(n, a);
    if (!rc && !front) rc = gather_rows(a, x, rows, 0.0f, 0, 0, nullptr, s);
    if (!rc) rc = forward_rows(n, a, front ? x : nullptr, nullptr, false, rows, s);
    c.order = a->ws.order;
    return rc ? rc : control_run(ctl, c, s);
}

}  // namespace

int adapters_create(const Net* n, uint32_t slots, uint32_t rank, float scale, const float* init, uint64_t seed, Adapters** out)
{
    Adapters* a = new (std::nothrow) Adapters();
    if (!a) { set_error("out of host memory"); return SZH_ENOMEM; }
    a->in = n->in; a->h1 = n->h1; a->h2 = n->h2; a->out = n->out;
    a->slots = slots; a->rank = rank; a->scale = scale; a->device = n->device;
    const uint64_t np = a->per_slot() * slots;
    hipError_t he = hipMalloc((void**)&a->d_params, (np + 1) * sizeof(float));
    if (he == hipSuccess) he = hipMalloc((void**)&a->d_grad, (np + 2ull * slots) * sizeof(float));
    if (he == hipSuccess) he = hipMalloc((void**)&a->d_sums, 2ull * slots * sizeof(double));
    if (he != hipSuccess) { adapters_destroy(a); return hip_fail(he, "adapter allocation"); }
    int rc = adapters_zero_grad(a, nullptr);
    if (!rc && init) rc = adapters_set_params(a, 0, slots, init);
    if (!rc && !init) {
        // A ~ U(-0.5, 0.5) / sqrt(its inputs), B = 0: a new adapter changes nothing until it is trained
        try {
            std::vector<float> p(np, 0.0f);
            const float s2 = 1.0f / std::sqrt((float)a->h1), s3 = 1.0f / std::sqrt((float)a->h2);
            for (uint32_t k = 0; k < slots; ++k) {
                float* q = p.data() + k * a->per_slot();
                for (uint64_t i = a->off_a2(); i < a->off_b2(); ++i) q[i] = s2 * init_uniform(seed, k * a->per_slot() + i);
                for (uint64_t i = a->off_a3(); i < a->off_b3(); ++i) q[i] = s3 * init_uniform(seed, k * a->per_slot() + i);
            }
            rc = adapters_set_params(a, 0, slots, p.data());
        } catch (const std::bad_alloc&) {
            set_error("out of host memory");
            rc = SZH_ENOMEM;
        }
    }
    if (!rc && hipDeviceSynchronize() != hipSuccess) { set_error("device synchronize failed"); rc = SZH_ENODEVICE; }
    if (rc) { adapters_destroy(a); return rc; }
    *out = a;
    return SZH_OK;
}

void adapters_destroy(Adapters* a)
{
    if (!a) return;
    clip_destroy(a->clip);
    if (a->d_params) (void)hipFree(a->d_params);
    if (a->d_grad) (void)hipFree(a->d_grad);
    if (a->d_sums) (void)hipFree(a->d_sums);
    for (char* p : a->arenas) (void)hipFree(p);
    delete a;
}

int adapters_set_params(Adapters* a, uint32_t slot0, uint32_t count, const float* flat)
{
    SZ_HIP(hipDeviceSynchronize());
    SZ_HIP(hipMemcpy(a->d_params + slot0 * a->per_slot(), flat, count * a->per_slot() * sizeof(float), hipMemcpyHostToDevice));
    return SZH_OK;
}

int adapters_get_params(Adapters* a, uint32_t slot0, uint32_t count, float* flat)
{
    SZ_HIP(hipDeviceSynchronize());
    SZ_HIP(hipMemcpy(flat, a->d_params + slot0 * a->per_slot(), count * a->per_slot() * sizeof(float), hipMemcpyDeviceToHost));
    return SZH_OK;
}

int adapters_reserve(Adapters* a, uint64_t rows, bool training)
{
    if (training)
        if (int rc = adapters_clip_tables(a)) return rc;
    return ensure(a, rows, training, nullptr);
}

int adapters_forward(Net* n, Adapters* a, const float* x, const int32_t* slots_dev, uint64_t rows, const Controls& ctl, float* logits,
                     float* probs, hipStream_t s)
{
    if (int rc = check_pair(n, a)) return rc;
    if (rows == 0 || n->out == 0) return SZH_OK;
    const uint64_t results = rows * n->out, feats = rows * n->in;
    if ((logits && probs && overlap(logits, results, probs, results)) || (logits && overlap(logits, results, x, feats)) ||
        (probs && overlap(probs, results, x, feats))) {
        set_error("logits, probabilities and features overlap");
        return SZH_EINVAL;
    }
    if (int rc = ensure(a, rows, false, s)) return rc;
    for (uint64_t r0 = 0; r0 < rows; r0 += kAdaptRows) {
        const uint32_t R = (uint32_t)std::min<uint64_t>(kAdaptRows, rows - r0);
        ControlRun c{};
        c.in = a->ws.lg; c.ld_in = a->ws.ld3; c.rows = R; c.classes = n->out;
        c.raw = logits ? logits + r0 * n->out : nullptr; c.ld_raw = n->out;
        c.out = probs ? probs + r0 * n->out : nullptr; c.ld_out = n->out; c.probs = true;
        if (int rc = infer_rows(n, a, x + r0 * n->in, slots_dev + r0, R, from_row(ctl, r0), c, s)) return rc;
    }
    return SZH_OK;
}

int adapters_vote(Net* n, Adapters* a, const float* x, const int32_t* slots_dev, uint64_t rows, const Controls& ctl, float threshold,
                  const int32_t* group, uint32_t groups, unsigned long long* counts, hipStream_t s)
{
    if (int rc = check_pair(n, a)) return rc;
    if (rows == 0 || n->out == 0) return SZH_OK;
    if (int rc = ensure(a, rows, false, s)) return rc;
    for (uint64_t r0 = 0; r0 < rows; r0 += kAdaptRows) {
        const uint32_t R = (uint32_t)std::min<uint64_t>(kAdaptRows, rows - r0);
        ControlRun c{};
        c.in = a->ws.lg; c.ld_in = a->ws.ld3; c.rows = R; c.classes = n->out;
        c.threshold = threshold; c.group = group ? group + r0 : nullptr; c.groups = groups; c.votes = counts;
        if (int rc = infer_rows(n, a, x + r0 * n->in, slots_dev + r0, R, from_row(ctl, r0), c, s)) return rc;
    }
    return SZH_OK;
}

int adapters_accumulate(Net* n, Adapters* a, const float* x, const int32_t* labels, const int32_t* slots_dev, uint64_t rows,
                        const Controls& ctl, float dropout, uint64_t seed, hipStream_t s)
{
    if (int rc = check_pair(n, a)) return rc;
    if (rows == 0 || n->out == 0) return SZH_OK;
    if (int rc = ensure(a, rows, true, s)) return rc;
    AdaptWorkspace& w = a->ws;
    const float* F = a->d_params;
    const int r = (int)a->rank, h2 = (int)n->h2, out = (int)n->out;
    for (uint64_t r0 = 0; r0 < rows; r0 += kAdaptRows) {
        const uint32_t R = (uint32_t)std::min<uint64_t>(kAdaptRows, rows - r0);
        int rc = group_rows(a, slots_dev + r0, R, s);
        const bool few = few_rows(n, R, true), front = !few && front_applies(n, a) && dropout <= 0.0f;
        if (!rc && !front) rc = gather_rows(a, x + r0 * n->in, R, dropout, seed, r0, w.live0, s);
        ControlRun c{};
        c.in = w.lg; c.ld_in = w.ld3; c.rows = R; c.classes = n->out; c.order = w.order;
        c.out = w.lg; c.ld_out = w.ld3; c.labels = labels + r0; c.row_live = w.live0; c.row_slot = w.row_slot; c.loss = w.loss; c.live = w.live;
        const Controls ctl_r = from_row(ctl, r0);
        if (!rc && few) rc = forward_few(n, a, w.xs, w.ldx, w.row_slot, R, ctl_r, c, w.u2, w.u3, s);
        const bool tail = !few && tail_applies(a);
        if (!rc && !few) rc = forward_rows(n, a, front ? x + r0 * n->in : nullptr, w.live0, tail, R, s);
        if (!rc && tail) rc = tail_rows(n, a, ctl_r, c, R, s);
        if (!rc && !few && !tail) rc = control_run(ctl_r, c, s);   // lg now holds d3
        if (rc) return rc;
        const bool back_done = tail || (few && (uint64_t)n->h2 * n->out <= kRowOutFloats);  // (by the row kernel)
        if (!back_done && back_applies(a)) {
            rc = back_rows(n, a, R, s);
            if (rc) return rc;
        } else if (!back_done) {
            rc = low_product(a, w.lg, w.ld3, out, F + a->off_b3(), 1, out, R, w.g3, s);
            if (rc) return rc;
            GemmArgs g{};
            g.A = w.lg; g.lda = w.ld3; g.B = n->d_params + n->off_w3(); g.ldb = out; g.C = w.d2; g.ldc = w.ld2;
            g.M = (int)R; g.N = h2; g.K = g.k_chunk = out; g.aux = w.h2; g.ldaux = w.ld2;
            adapt_args(g, a, w.g3, F + a->off_a3(), 1, r);
            rc = launch_gemm_rows<A_ROWS, B_ROWS, EPI_ADAPT_DTANH, T_ADAPT_D2, 64>(g, s);  // (a short k, as above)
            if (!rc) rc = low_product(a, w.d2, w.ld2, h2, F + a->off_b2(), 1, h2, R, w.g2, s);
            if (rc) return rc;
        }
        rc = factor_gradients(a, R, s);
        if (rc) return rc;
    }
    return SZH_OK;
}

int adapters_zero_grad(Adapters* a, hipStream_t s)
{
    const uint64_t n = (a->per_slot() + 2) * a->slots;
    hipLaunchKernelGGL(adapter_clear_kernel, dim3((unsigned)std::min<uint64_t>((n + 1023) / 1024, 4096)), dim3(256), 0, s, a->d_grad, n, a->d_sums,
                       2ull * a->slots);
    SZ_HIP(hipGetLastError());
    return SZH_OK;
}

int adapters_clip(Adapters* a, float max_norm, float* norms_dev, hipStream_t s)
{
    if (!a->clip) {
        if (capturing(s)) { set_error("adapters: the first clipping allocates its tables and cannot be captured (szh_adapters_reserve makes them)"); return SZH_EINVAL; }
        if (int rc = adapters_clip_tables(a)) return rc;
    }
    return clip_run(a->clip, max_norm, norms_dev, s);
}

int adapters_clip_tables(Adapters* a)
{
    if (a->clip) return SZH_OK;
    std::vector<ClipTensor> t(a->slots);
    for (uint32_t k = 0; k < a->slots; ++k) t[k] = {a->d_grad + k * a->per_slot(), a->d_grad + k * a->per_slot(), a->per_slot(), k};
    return clip_create(t.data(), a->slots, a->slots, a->d_grad + a->per_slot() * a->slots + 1, 2, &a->clip);
}

int adapters_apply(Adapters* a, float lr, hipStream_t s)
{
    ProfScope prof("apply", s);
    hipLaunchKernelGGL(adapter_apply_kernel, dim3((unsigned)((a->per_slot() + 255) / 256), a->slots), dim3(256), 0, s, a->d_params, a->d_grad,
                       a->d_grad + a->per_slot() * a->slots, a->per_slot(), lr);
    SZ_HIP(hipGetLastError());
    return SZH_OK;
}

}  // namespace sz
