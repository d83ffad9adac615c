// The gated MLP block in training: forward with what its gradients need kept, and the gradients.
//
//   a = x W1, b = x W3, h = silu(a) b, y = h W2
//   dh = dy W2^T,  da = dh b silu'(a),  db = dh silu(a)      silu'(a) = s + a s (1 - s),  s = 1 / (1 + exp(-a))
//   dx = da W1^T + db W3^T,  dW1 = x^T da,  dW3 = x^T db,  dW2 = h^T dy
//
// Four launches (two more that add up partial results where there are few rows): both first products with the activation in their epilogue;
// y; dh, whose epilogue reads a and b and writes da and db, so that dh is never written; and dx with all three weight gradients. a and b are
// kept in 32 bits: rounded to bf16 they would put two more roundings into da, beside its own, and the gradients' error from 1.4 to 1.8 times
// that of the result's rounding; h, da and db are rounded to bf16 because the tensor cores multiply bf16.
// 8192 rows, 4096 x 14336 x 4096, forward and backward: 7.0 to 7.2 ms at the power limit (1.21 to 1.24 PFLOP/s), 5.9 ms as single launches from idle;
// 64 rows: 281 to 301 us, 2.4 TB/s of weights and gradients, bound by the loads in flight and by two rounds of tiles over 74 pairs of SMs.
// Matrices whose rows are no whole 16 bytes are copied, two bytes a thread and turn: 64 rows, 4095 x 14335 x 4095: 2.33 ms; 1777 rows, 1023 x 2815 x 1023: 293 us,
// where 1024 x 2816 x 1024 takes 122.
#include "train_common.cuh"

namespace mimk {

namespace {

using namespace group;

constexpr int64_t LIM = int64_t(1) << 30;

// The buffer kept from the forward pass to the backward one: a and b as f32, h as bf16, rows of `pitch` elements.
struct Kept {
    int64_t pitch;
    float *a, *b;
    __nv_bfloat16* h;
    size_t bytes;
};
Kept kept_layout(const mimk_mlp_train_desc& d) {
    Space space(d.kept);
    Kept k;
    k.pitch = up(d.f, 8);
    const size_t cells = size_t(d.m) * size_t(k.pitch);
    k.a = static_cast<float*>(space.take(cells * 4)), k.b = static_cast<float*>(space.take(cells * 4));
    k.h     = static_cast<__nv_bfloat16*>(space.take(cells * 2));
    k.bytes = space.used();
    return k;
}

int blocks_of(int64_t k) { return int((k + BK - 1) / BK); }

struct Plan {
    Staged x, w1, w3, w2;
    Staged y;                   // forward
    Staged dy, dx, dw1, dw3, dw2;  // backward
    void *da, *db;
    float* part;  // partial results of y, or of dx
    int64_t pitch, part_pitch, rows_pad;
    int splits;
};

Plan plan(const mimk_mlp_train_desc& d, bool backward, Space& space, int sm_count) {
    Plan p{};
    const bool nk = d.b_layout == MIMK_B_NK;
    auto weight   = [&](const void* w, int64_t in, int64_t out) { return nk ? stage(space, w, out, in) : stage(space, w, in, out); };
    p.x = stage(space, d.x, d.m, d.k);
    p.w1 = weight(d.w1, d.k, d.f), p.w3 = weight(d.w3, d.k, d.f), p.w2 = weight(d.w2, d.f, d.n);
    const int64_t n  = backward ? d.k : d.n;  // columns of the product whose k-blocks may be dealt out
    const int64_t kb = (backward ? 2 : 1) * int64_t(blocks_of(d.f));
    p.splits         = pick_splits(d.m, n, kb, sm_count);
    p.rows_pad       = up(d.m, 32);
    p.part_pitch     = up(n, 4);
    if (p.splits > 1) p.part = static_cast<float*>(space.take(size_t(p.splits) * size_t(p.rows_pad) * size_t(p.part_pitch) * 4));
    if (!backward) {
        p.y = stage(space, d.y, d.m, d.n);
        return p;
    }
    p.dy = stage(space, d.dy, d.m, d.n), p.dx = stage(space, d.dx, d.m, d.k);
    p.dw1 = weight(d.dw1, d.k, d.f), p.dw3 = weight(d.dw3, d.k, d.f), p.dw2 = weight(d.dw2, d.f, d.n);
    p.pitch = up(d.f, 8);
    p.da = space.take(size_t(d.m) * size_t(p.pitch) * 2), p.db = space.take(size_t(d.m) * size_t(p.pitch) * 2);
    return p;
}

int check(const mimk_mlp_train_desc* d) {
    if (!d) return MIMK_E_ARG;
    if (d->m < 0 || d->k < 0 || d->f < 0 || d->n < 0) return MIMK_E_ARG;
    if (d->dtype != MIMK_BF16) return MIMK_E_DTYPE;
    if (d->b_layout != MIMK_B_KN && d->b_layout != MIMK_B_NK) return MIMK_E_ARG;
    if (d->m >= LIM || d->k >= LIM || d->f >= LIM || d->n >= LIM) return MIMK_E_UNSUPPORTED;
    return MIMK_OK;
}
bool nothing(const mimk_mlp_train_desc& d) { return d.m == 0 || d.k == 0 || d.f == 0 || d.n == 0; }
int zero(void* p, int64_t rows, int64_t cols, cudaStream_t s) {
    if (rows && cols) {
        if (!p) return MIMK_E_ARG;
        MIMK_CUDA_TRY(cudaMemsetAsync(p, 0, size_t(rows) * size_t(cols) * 2, s));
    }
    return MIMK_OK;
}

Problem problem(int64_t m, int64_t n, int64_t k, bool a_mn, bool b_mn) {
    Problem p{};
    p.M = int(m), p.N = int(n), p.kb[0] = blocks_of(k), p.a_mn = a_mn, p.b_mn = b_mn, p.splits = 1;
    return p;
}
// the result of a STORE problem: bf16 where it belongs, or f32 partial ones
int store_to(Problem& pr, CUtensorMap* map, const Plan& p, const Mat& out) {
    if (p.splits == 1) return result_map(map, const_cast<void*>(out.p), false, out.rows, out.cols, out.pitch);
    pr.splits = p.splits, pr.rows_pad = int(p.rows_pad), pr.out_f32 = 1;
    return result_map(map, p.part, true, p.splits * p.rows_pad, out.cols, p.part_pitch);
}

}  // namespace
}  // namespace mimk

using namespace mimk;

extern "C" int mimk_mlp_gated_train_sizes(const mimk_mlp_train_desc* d, uint64_t* kept, uint64_t* forward, uint64_t* backward) {
    MIMK_TRY(check(d));
    int st                = MIMK_OK;
    const DeviceInfo* dev = device_info(&st);
    if (!dev) return st;
    mimk_mlp_train_desc sized = *d;
    sized.kept                = nullptr;
    if (kept) *kept = kept_layout(sized).bytes;
    for (int b = 0; b < 2; ++b) {
        Space space(nullptr);
        plan(*d, b != 0, space, dev->sm_count);
        if (uint64_t* out = b ? backward : forward) *out = nothing(*d) ? 0 : space.used();
    }
    return MIMK_OK;
}

extern "C" int mimk_mlp_gated_fwd(const mimk_mlp_train_desc* d, void* stream) {
    MIMK_TRY(check(d));
    int st                = MIMK_OK;
    const DeviceInfo* dev = device_info(&st);
    if (!dev) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (nothing(*d)) return zero(d->y, d->m, d->n, s);
    if (!d->x || !d->w1 || !d->w3 || !d->w2 || !d->y || !d->kept) return MIMK_E_ARG;
    if (!aligned16(d->kept)) return MIMK_E_ALIGN;
    Space space(d->workspace);
    const Plan p = plan(*d, false, space, dev->sm_count);
    if (space.used() > d->workspace_bytes || (space.used() && !d->workspace)) return MIMK_E_WORKSPACE;
    if (space.used() && !aligned16(d->workspace)) return MIMK_E_ALIGN;
    const Kept kept = kept_layout(*d);
    const bool mn   = d->b_layout == MIMK_B_KN;
    for (const Staged* x : {&p.x, &p.w1, &p.w3, &p.w2}) MIMK_TRY(stage_in(*x, s));

    Maps maps;
    Args args{};
    args.count = 1, args.status = dev->status_dev;
    args.p[0] = problem(d->m, d->f, d->k, false, mn);
    MIMK_TRY(operand_map(&maps.a[0][0], p.x.use, false, BM));
    MIMK_TRY(operand_map(&maps.b[0][0], p.w1.use, mn, 64));
    MIMK_TRY(operand_map(&maps.b[0][1], p.w3.use, mn, 64));
    MIMK_TRY(result_map(&maps.out[0], kept.h, false, d->m, d->f, kept.pitch));
    MIMK_TRY(result_map(&maps.extra[0], kept.a, true, d->m, d->f, kept.pitch));
    MIMK_TRY(result_map(&maps.extra[1], kept.b, true, d->m, d->f, kept.pitch));
    MIMK_TRY(launch_group<GATED_FWD>(maps, args, *dev, s));

    const Mat h = {kept.h, d->m, d->f, kept.pitch};
    args.p[0]   = problem(d->m, d->n, d->f, false, mn);
    MIMK_TRY(operand_map(&maps.a[0][0], h, false, BM));
    MIMK_TRY(operand_map(&maps.b[0][0], p.w2.use, mn, 128));
    MIMK_TRY(store_to(args.p[0], &maps.out[0], p, p.y.use));
    MIMK_TRY(launch_group<STORE>(maps, args, *dev, s));
    if (p.splits > 1) return sum_parts(p.part, p.splits, p.rows_pad, p.part_pitch, d->y, d->n, d->m, d->n, s);
    return stage_out(p.y, s);
}

extern "C" int mimk_mlp_gated_bwd(const mimk_mlp_train_desc* d, void* stream) {
    MIMK_TRY(check(d));
    int st                = MIMK_OK;
    const DeviceInfo* dev = device_info(&st);
    if (!dev) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (nothing(*d)) {
        MIMK_TRY(zero(d->dx, d->m, d->k, s));
        MIMK_TRY(zero(d->dw1, d->k, d->f, s));
        MIMK_TRY(zero(d->dw3, d->k, d->f, s));
        return zero(d->dw2, d->f, d->n, s);
    }
    if (!d->x || !d->w1 || !d->w3 || !d->w2 || !d->kept || !d->dy || !d->dx || !d->dw1 || !d->dw3 || !d->dw2) return MIMK_E_ARG;
    if (!aligned16(d->kept)) return MIMK_E_ALIGN;
    Space space(d->workspace);
    const Plan p = plan(*d, true, space, dev->sm_count);
    if (space.used() > d->workspace_bytes || !d->workspace) return MIMK_E_WORKSPACE;
    if (!aligned16(d->workspace)) return MIMK_E_ALIGN;
    const Kept kept = kept_layout(*d);
    const bool nk   = d->b_layout == MIMK_B_NK;
    for (const Staged* x : {&p.x, &p.w1, &p.w3, &p.w2, &p.dy}) MIMK_TRY(stage_in(*x, s));

    Maps maps;
    Args args{};
    args.count = 1, args.status = dev->status_dev;
    const Mat da = {p.da, d->m, d->f, p.pitch}, db = {p.db, d->m, d->f, p.pitch}, h = {kept.h, d->m, d->f, kept.pitch};
    // dh = dy W2^T, and da and db from it. W2 [f, n] has its K axis contiguous here, W2 stored [n, f] its N axis.
    args.p[0] = problem(d->m, d->f, d->n, false, nk);
    MIMK_TRY(operand_map(&maps.a[0][0], p.dy.use, false, BM));
    MIMK_TRY(operand_map(&maps.b[0][0], p.w2.use, nk, 128));
    MIMK_TRY(result_map(&maps.extra[0], kept.a, true, d->m, d->f, kept.pitch));
    MIMK_TRY(result_map(&maps.extra[1], kept.b, true, d->m, d->f, kept.pitch));
    MIMK_TRY(result_map(&maps.out[0], p.da, false, d->m, d->f, p.pitch));
    MIMK_TRY(result_map(&maps.out[1], p.db, false, d->m, d->f, p.pitch));
    MIMK_TRY(launch_group<GATED_BWD>(maps, args, *dev, s));

    // dx = da W1^T + db W3^T first, whose tiles are the longest where there are more hidden columns than rows
    args.count     = 4;
    args.p[0]      = problem(d->m, d->k, d->f, false, nk);
    args.p[0].kb[1] = args.p[0].kb[0];
    MIMK_TRY(operand_map(&maps.a[0][0], da, false, BM));
    MIMK_TRY(operand_map(&maps.a[0][1], db, false, BM));
    MIMK_TRY(operand_map(&maps.b[0][0], p.w1.use, nk, 128));
    MIMK_TRY(operand_map(&maps.b[0][1], p.w3.use, nk, 128));
    MIMK_TRY(store_to(args.p[0], &maps.out[0], p, p.dx.use));
    // the weights' gradients, in the weights' own layout: x^T da or its transpose da^T x
    const Mat* left[3]      = {nk ? &da : &p.x.use, nk ? &db : &p.x.use, nk ? &p.dy.use : &h};
    const Mat* right[3]     = {nk ? &p.x.use : &da, nk ? &p.x.use : &db, nk ? &h : &p.dy.use};
    const Staged* result[3] = {&p.dw1, &p.dw3, &p.dw2};
    for (int i = 0; i < 3; ++i) {
        const Mat& out  = result[i]->use;
        args.p[i + 1] = problem(out.rows, out.cols, d->m, true, true);
        MIMK_TRY(operand_map(&maps.a[i + 1][0], *left[i], true, BM));
        MIMK_TRY(operand_map(&maps.b[i + 1][0], *right[i], true, 128));
        MIMK_TRY(result_map(&maps.out[i + 1], const_cast<void*>(out.p), false, out.rows, out.cols, out.pitch));
    }
    MIMK_TRY(launch_group<STORE>(maps, args, *dev, s));
    for (const Staged* x : result) MIMK_TRY(stage_out(*x, s));
    if (p.splits > 1) return sum_parts(p.part, p.splits, p.rows_pad, p.part_pitch, d->dx, d->k, d->m, d->k, s);
    return stage_out(p.dx, s);
}
