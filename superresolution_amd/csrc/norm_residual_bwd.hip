// Backward of the fused block norm: the C entry, how rows are cut into work, and the launch that adds what the row kernels
// (norm_residual_bwd.h) leave.
#include "norm_residual_bwd.h"

using namespace srhip_norm;

namespace {

// Adds the sums of work-groups and items: 32 columns to a block, 32 thread groups taking every 32nd sum, then theirs in
// order.  Block b: section b / cblocks (0, 1: dw_pre, db_pre; 2, 3: dw_post, db_post; 4: ds; 5 + i: gate i) of 32 channels.  A
// launch has fewer than 2^32 threads along x: gates beyond kMaxBlocks lie along y, `gate_row` to each of its rows.
// A chain of dependent-looking loads is what bounds it: a thousand sums in 32 steps of eight loads each (4.6 MB; 64 columns and
// 16 groups, with a division by the items of a gate in every step, took 34 us for 64 channels, this 5).
constexpr int kCols = 32, kParts = 32;
constexpr long long kMaxBlocks = (1ll << 32) / (kCols * kParts) - 1;
__global__ __launch_bounds__(kCols * kParts) void norm_residual_bwd_sums_kernel(const NormBwdParams p, const int nwg, const int cblocks, const long long gates, const long long gate_row)
{
    __shared__ float red[2][kParts][kCols];
    const int col = threadIdx.x % kCols, part = threadIdx.x / kCols;
    const int section = (int)(blockIdx.x / (unsigned)cblocks);
    const int ch = (int)(blockIdx.x % (unsigned)cblocks) * kCols + col;
    const bool in = ch < p.c;
    const long long gate = section - 5 + blockIdx.y * gate_row;
    if (section < 5 ? blockIdx.y != 0 : gate >= gates) return;   // uniform over the block, as all that follow
    const float scale = p.scale_ptr ? *p.scale_ptr : p.scale;
    float a = 0.0f, b = 0.0f;
    if (section < 2) {
        float* dst = section == 0 ? p.dpre_w : p.dpre_b;
        if (dst == nullptr) return;
        if (in) {
            const float* src = p.wg_sums + section * p.c + ch;
#pragma unroll 8
            for (int k = part; k < nwg; k += kParts) a += src[2ll * k * p.c];
        }
    } else if (section < 4) {
        float* dst = section == 2 ? p.dpost_w : p.dpost_b;
        if (dst == nullptr) return;
        if (in) {
            const float* src = p.item_sums + (section - 2) * p.c + ch;
            if (p.gate_mode == SRHIP_GATE_ROWS && p.items > p.segs) {
                // several gates: each item's sum times its gate
                long long s = part / p.segs;
                int rem = part % p.segs;
                const int s_step = kParts / p.segs, r_step = kParts % p.segs;
#pragma unroll 8
                for (long long k = part; k < p.items; k += kParts) {
                    float slope;
                    a += gate_value(p, s, ch, slope) * src[2 * k * p.c];
                    s += s_step;
                    rem += r_step;
                    if (rem >= p.segs) { rem -= p.segs; ++s; }
                }
            } else {
#pragma unroll 8
                for (long long k = part; k < p.items; k += kParts) a += src[2 * k * p.c];
                float slope;
                a *= gate_value(p, 0, ch, slope);
            }
        }
    } else if (section == 4) {
        if (p.dscale == nullptr || blockIdx.x % (unsigned)cblocks != 0) return;
#pragma unroll 4
        for (long long k = threadIdx.x; k < p.items; k += kCols * kParts) a += p.item_scale[k];
    } else {
        if (in) {
            const float* src = p.item_sums + gate * p.segs * 2 * p.c + ch;
#pragma unroll 8
            for (int k = part; k < p.segs; k += kParts) {
                a += src[2ll * k * p.c];
                b += src[(2ll * k + 1) * p.c];
            }
        }
    }
    red[0][part][col] = a;
    red[1][part][col] = b;
    __syncthreads();
    if (part != 0) return;
#pragma unroll
    for (int k = 1; k < kParts; ++k) { a += red[0][k][col]; b += red[1][k][col]; }
    if (section == 4) {
        a = lanes_sum<kCols>(a);
        if (col == 0) *p.dscale = a;
        return;
    }
    if (!in) return;
    if (section < 2) (section == 0 ? p.dpre_w : p.dpre_b)[ch] = a;
    else if (section < 4) (section == 2 ? p.dpost_w : p.dpost_b)[ch] = scale * a;
    else {
        float slope;
        gate_value(p, gate, ch, slope);
        ((float*)p.dgate)[gate * p.c + ch] = gate_gradient(p, ch, scale * slope, a, b);
    }
}

int rows(const srhip_norm_residual_bwd_args* a, const NormBwdParams* p, Plan& q, hipStream_t stream)
{
    const bool ck = a->h_scales || a->r_scales, mapg = a->gate_mode == SRHIP_GATE_MAP;
    if (a->dtype == SRHIP_DT_BF16) return (a->c % 8 ? rows_bf16_odd : rows_bf16)(a->c, ck, mapg, p, q, stream);
    return (a->c % 4 ? rows_f32_odd : rows_f32)(a->c, ck, mapg, p, q, stream);
}

// Items and work-groups: a function of the shapes and types alone (and of the device), so that the workspace can be sized before
// the call.
Plan plan_of(const srhip_norm_residual_bwd_args* a)
{
    Plan q;
    rows(a, nullptr, q, nullptr);
    const long long passes = (a->rows + q.rpb - 1) / q.rpb;
    const long long cus = srhip_num_cus(), resident = cus * q.grid;
    // A work-group's sums (4 c floats written, and read again) weigh as much as one or two of its rows: eight passes to a
    // work-group at least, once every CU has one.
    long long grid = passes / 8;
    if (grid < cus) grid = passes < cus ? passes : cus;
    if (passes <= 4) grid = 1;   // a few rows: one work-group and no second launch (four fp32 rows of 1024: 20.5 us a call, with two 24)
    if (grid > resident) grid = resident;
    const long long gates = a->gate_mode == SRHIP_GATE_ROWS ? a->rows / a->rows_per_gate : 1;
    const long long per_gate = a->rows / gates;
    // Items run in rounds of `grid`, and a round of a few takes as long as a full one: as many items to a gate as r rounds hold, for
    // the r of the fewest or three more that takes the least passes (an item's sums counted as two), and a further round for a
    // thirty-second at least.  (64 channels from checkpoints, 1024 work-groups at once: three crops of 1024^2 in 1026 items 614 us, in
    // 1023 428; seven in 1029 1417, in 1022 983; 600 gates of 3500 rows in 1200 items 389, in 3000 323.)
    const long long passes_per_gate = (per_gate + q.rpb - 1) / q.rpb, fewest = (gates + grid - 1) / grid;
    long long segs = 1, least = -1;
    for (long long r = fewest; r < fewest + 4; ++r) {
        long long k = r * grid / gates;
        if (k > passes_per_gate) k = passes_per_gate;
        const long long cost = r * ((passes_per_gate + k - 1) / k + 2);
        if (least < 0 || cost < least - least / 32) { least = cost; segs = k; }
    }
    q.seg_rows = (((per_gate + segs - 1) / segs) + q.rpb - 1) / q.rpb * q.rpb;
    q.segs = (int)((per_gate + q.seg_rows - 1) / q.seg_rows);
    q.items = gates * q.segs;
    q.grid = (int)(q.items < grid ? q.items : grid);
    return q;
}

}  // namespace

static int bad_shape(const srhip_norm_residual_bwd_args* a)
{
    SRHIP_REQUIRE(a, "norm_residual_bwd: null pointer");
    SRHIP_REQUIRE(a->rows >= 0 && a->c >= 1 && a->c <= SRHIP_NORM_MAX_C, "norm_residual_bwd: bad shape (%lld rows of %d channels; 1 .. %d channels)", a->rows, a->c, SRHIP_NORM_MAX_C);
    SRHIP_REQUIRE(a->gate_mode >= SRHIP_GATE_NONE && a->gate_mode <= SRHIP_GATE_MAP, "norm_residual_bwd: unknown gate mode %d", a->gate_mode);
    SRHIP_REQUIRE(a->rows == 0 || a->gate_mode != SRHIP_GATE_ROWS || (a->rows_per_gate >= 1 && a->rows % a->rows_per_gate == 0), "norm_residual_bwd: %lld rows are not a multiple of %lld rows per gate", a->rows, a->rows_per_gate);
    return SRHIP_OK;
}

extern "C" {

SRHIP_API size_t srhip_norm_residual_bwd_workspace_bytes(const srhip_norm_residual_bwd_args* a)
{
    if (bad_shape(a) != SRHIP_OK || a->rows == 0) return 0;
    const Plan q = plan_of(a);
    return ((size_t)q.grid * 2 * a->c + (size_t)q.items * (2 * (size_t)a->c + 1)) * sizeof(float);
}

SRHIP_API int srhip_norm_residual_bwd(const srhip_norm_residual_bwd_args* a, void* stream)
{
    const int rc = bad_shape(a);
    if (rc != SRHIP_OK) return rc;
    SRHIP_REQUIRE(a->dtype == SRHIP_DT_BF16 || a->dtype == SRHIP_DT_F32, "norm_residual_bwd: unknown type %d", a->dtype);
    SRHIP_REQUIRE(a->kind == SRHIP_NORM_LAYER || a->kind == SRHIP_NORM_RMS, "norm_residual_bwd: unknown norm %d", a->kind);
    SRHIP_REQUIRE(a->eps >= 0.0f, "norm_residual_bwd: eps must not be negative");
    SRHIP_REQUIRE(a->rows >= 1, "norm_residual_bwd: no rows");
    SRHIP_REQUIRE(a->dx && (a->dr || a->pre), "norm_residual_bwd: null pointer");
    SRHIP_REQUIRE(!a->pre || (a->r && a->dn && a->pre_weight && a->dpre_weight), "norm_residual_bwd: the norm behind the sum needs r, dn, its weight and room for its gradient");
    SRHIP_REQUIRE(a->dh || (!a->post && a->gate_mode == SRHIP_GATE_NONE && !a->dscale), "norm_residual_bwd: a gate, a scale or a post norm without a branch");
    SRHIP_REQUIRE(!a->post || (a->post_weight && a->dpost_weight), "norm_residual_bwd: the post norm needs its weight and room for its gradient");
    SRHIP_REQUIRE(a->gate_mode == SRHIP_GATE_NONE || (a->gate && a->dgate), "norm_residual_bwd: null gate");
    const int need_h = a->dh && (a->post || a->gate_mode != SRHIP_GATE_NONE || a->dscale);
    SRHIP_REQUIRE(!need_h || a->h, "norm_residual_bwd: null branch");
    SRHIP_REQUIRE(a->workspace, "norm_residual_bwd: null workspace");
    Plan q = plan_of(a);
    NormBwdParams p;
    p.h = (const char*)a->h; p.r = (const char*)a->r; p.dr = (const char*)a->dr; p.dn = (const char*)a->dn; p.gate = (const char*)a->gate;
    p.h_scales = (const unsigned char*)a->h_scales; p.r_scales = (const unsigned char*)a->r_scales;
    p.post_w = a->post ? a->post_weight : nullptr; p.post_b = a->post ? a->post_bias : nullptr; p.pre_w = a->pre ? a->pre_weight : nullptr;
    p.scale_ptr = a->scale_ptr;
    p.dx = (char*)a->dx; p.dh = (char*)a->dh; p.dgate = (char*)a->dgate;
    p.wg_sums = (float*)a->workspace;
    p.item_sums = p.wg_sums + (size_t)q.grid * 2 * a->c;
    p.item_scale = p.item_sums + (size_t)q.items * 2 * a->c;
    p.dpost_w = a->post ? a->dpost_weight : nullptr; p.dpost_b = a->post ? a->dpost_bias : nullptr;
    p.dpre_w = a->pre ? a->dpre_weight : nullptr; p.dpre_b = a->pre ? a->dpre_bias : nullptr;
    p.dscale = a->dscale;
    p.rows = a->rows;
    p.rows_per_gate = a->gate_mode == SRHIP_GATE_ROWS ? a->rows_per_gate : a->rows;
    p.seg_rows = q.seg_rows; p.items = q.items; p.segs = q.segs;
    p.c = a->c; p.groups = srhip_div_up(a->c, kCk8Group); p.layer = a->kind == SRHIP_NORM_LAYER; p.post = a->post; p.pre = a->pre;
    p.gate_mode = a->gate_mode; p.gate_f32 = a->dtype != SRHIP_DT_F32 && a->gate_f32; p.sigmoid = a->gate_sigmoid;
    p.need_h = need_h; p.item_flush = a->dh && (a->post || a->gate_mode == SRHIP_GATE_ROWS || a->dscale);
    p.scale = a->scale; p.eps = a->eps; p.inv_c = 1.0f / (float)a->c;
    const long long gates = p.gate_mode == SRHIP_GATE_ROWS ? a->rows / p.rows_per_gate : 0;
    const hipStream_t s = (hipStream_t)stream;
    const int cblocks = srhip_div_up(p.c, kCols);
    const long long most = kMaxBlocks / cblocks - 5, gate_row = gates < most ? gates : most;
    const long long gate_rows = gates > gate_row ? (gates + gate_row - 1) / gate_row : 1;
    SRHIP_REQUIRE(gate_rows < (1ll << 16), "norm_residual_bwd: too many gates");
    const int launched = rows(a, &p, q, s);
    if (launched != SRHIP_OK || q.items == 1 || (!p.pre && !p.item_flush)) return launched;
    hipLaunchKernelGGL(norm_residual_bwd_sums_kernel, dim3((unsigned)((5 + gate_row) * cblocks), (unsigned)gate_rows), dim3(kCols * kParts), 0, s, p, q.grid,
                       cblocks, gates, gate_row);
    return srhip_check_launch("norm_residual_bwd_sums_kernel");
}

}  // extern "C"
