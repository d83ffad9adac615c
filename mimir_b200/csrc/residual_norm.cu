// From one block of a model to the next, and its gradients:
//   u = e h post_gamma,  r_out = a r + b gate u,  x = s r_out gamma         e = 1 / sqrt(mean h^2 + eps),  s = 1 / sqrt(mean r_out^2 + eps)
//   t = dx gamma,  D = dr_out + s t - s^3 r_out mean(t r_out):  dr = a D,  dgamma = sum dx s r_out,  dgate = sum b u D
//   q = b gate post_gamma:  dpost_gamma = sum b gate e h D,  dh = e q D - e^3 h mean(q h D)
// A row belongs to a team of threads, a warp or a block, and stays in their registers. The backward pass has one join of sums for a row: with hats for
// e h and s r_out, and D = (dr_out + s t) - k r_out^,  k = s mean(t r_out^),  the second mean is mean(q h^ (dr_out + s t)) - k mean(q h^ r_out^). r_out is
// computed over again from r and h, the same bytes as reading it, so that a stream kept in bf16 is not rounded on the way into the gradients.
// Gradients over rows are summed by each block over its rows, in registers, and over the blocks by a second launch.
// What bounds it: the bytes.
#include "elements.cuh"
#include "train_common.cuh"

namespace mimk {

namespace {

constexpr int64_t MOST_COLUMNS = 32768, LIM = int64_t(1) << 31;

// A vector of d factors, f32 or bf16; absent: ones.
struct Factors {
    const void* p;
    int bf16;
};
template <int VEC>
__device__ __forceinline__ void factors_at(const Factors& f, int64_t at, float (&v)[VEC]) {
    if (!f.p) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = 1.f;
    } else if (f.bf16) {
        Run<__nv_bfloat16, VEC> r;
        r.load(static_cast<const __nv_bfloat16*>(f.p) + at), r.get(v);
    } else {
        Run<float, VEC> r;
        r.load(static_cast<const float*>(f.p) + at), r.get(v);
    }
}

template <class RT, class HT>
struct Args {
    int64_t n, d, gate_rows;
    const RT* r;
    const HT* h;
    Factors gamma, post_gamma, gate;
    RT* r_out;
    HT* x;
    float* kept;  // e of every row, then s
    const RT* dr_out;
    const HT* dx;
    RT* dr;
    HT* dh;
    // sums over rows: one row of d for each block, or (gate) for each unit of rows; a unit that is a whole group of the gate's writes dgate
    float *part_gamma, *part_post, *part_gate;
    void* dgate;
    int64_t groups, pieces;
    float eps, a, b;
};

// Sums of N values over a team: a warp, or a block.
template <int N>
__device__ __forceinline__ void team_sum(float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
    if (blockDim.x == 32) return;
    __shared__ float part[32][N];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    __syncthreads();  // (of an earlier call's reads)
    if (lane == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) part[warp][i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(lane < warps ? part[lane][i] : 0.f);
}

// VEC elements side by side, CH times, blockDim.x threads apart: what a thread holds of a row.
template <class RT, class HT, int VEC, int CH, int MAXT>
__global__ void __launch_bounds__(MAXT, 1) forward_kernel(const __grid_constant__ Args<RT, HT> g) {
    after_previous();
    const float per = 1.f / float(g.d);
    for (int64_t row = int64_t(blockIdx.x) * blockDim.y + threadIdx.y; row < g.n; row += int64_t(gridDim.x) * blockDim.y) {
        Run<RT, VEC> rr[CH];
        Run<HT, VEC> hr[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int64_t at = (c * int(blockDim.x) + int(threadIdx.x)) * VEC;
            rr[c].clear(), hr[c].clear();
            if (at < g.d) {
                rr[c].load(g.r + row * g.d + at);
                if (g.h) hr[c].load(g.h + row * g.d + at);
            }
        }
        float e = 1.f, sum[1];
        if (g.post_gamma.p) {
            sum[0] = 0.f;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                float h[VEC];
                hr[c].get(h);
#pragma unroll
                for (int j = 0; j < VEC; ++j) sum[0] = fmaf(h[j], h[j], sum[0]);
            }
            team_sum(sum);
            e = 1.f / sqrtf(sum[0] * per + g.eps);
        }
        const int64_t group = g.gate.p ? row / g.gate_rows : 0;
        float v[CH][VEC];
        sum[0] = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int64_t at = (c * int(blockDim.x) + int(threadIdx.x)) * VEC;
            rr[c].get(v[c]);
            if (at < g.d && g.h) {
                float h[VEC], f[VEC], q[VEC];
                hr[c].get(h);
                factors_at(g.post_gamma, at, f), factors_at(g.gate, group * g.d + at, q);
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[c][j] = fmaf(g.a, v[c][j], g.b * q[j] * (h[j] * e * f[j]));
                if (g.r_out) put(g.r_out + row * g.d + at, v[c]);
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) sum[0] = fmaf(v[c][j], v[c][j], sum[0]);
        }
        float s = 1.f;
        if (g.gamma.p) {
            team_sum(sum);
            s = 1.f / sqrtf(sum[0] * per + g.eps);
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int64_t at = (c * int(blockDim.x) + int(threadIdx.x)) * VEC;
                if (at >= g.d) break;
                float f[VEC];
                factors_at(g.gamma, at, f);
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[c][j] *= s * f[j];
                put(g.x + row * g.d + at, v[c]);
            }
        }
        if (g.kept && threadIdx.x == 0) g.kept[row] = e, g.kept[g.n + row] = s;
    }
}

template <class RT, class HT, int VEC, int CH, int MAXT>
__global__ void __launch_bounds__(MAXT, 1) backward_kernel(const __grid_constant__ Args<RT, HT> g) {
    after_previous();
    const float per   = 1.f / float(g.d);
    const int64_t team = int64_t(blockIdx.x) * blockDim.y + threadIdx.y, teams = int64_t(gridDim.x) * blockDim.y;
    float dgamma[CH][VEC] = {}, dpost[CH][VEC] = {};
    for (int64_t unit = team; unit < g.groups * g.pieces; unit += teams) {
        const int64_t group = unit / g.pieces, piece = unit - group * g.pieces, end = min(g.n, (group + 1) * g.gate_rows);
        float dgate[CH][VEC] = {};
        for (int64_t row = group * g.gate_rows + piece; row < end; row += g.pieces) {
            Run<RT, VEC> rr[CH], drr[CH];
            Run<HT, VEC> hr[CH], dxr[CH];
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int64_t at = (c * int(blockDim.x) + int(threadIdx.x)) * VEC, p = row * g.d + at;
                rr[c].clear(), drr[c].clear(), hr[c].clear(), dxr[c].clear();
                if (at < g.d) {
                    rr[c].load(g.r + p);
                    if (g.h) hr[c].load(g.h + p);
                    if (g.dr_out) drr[c].load(g.dr_out + p);
                    if (g.dx) dxr[c].load(g.dx + p);
                }
            }
            const float e = g.post_gamma.p ? g.kept[row] : 1.f, s = g.gamma.p ? g.kept[g.n + row] : 1.f;
            float sum[3] = {};
            float hat[CH][VEC], rhat[CH][VEC], before[CH][VEC], q[CH][VEC];  // h^, r_out^, dr_out + s t, q
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int64_t at = (c * int(blockDim.x) + int(threadIdx.x)) * VEC;
                float w[VEC], gate[VEC], dx[VEC];
                rr[c].get(rhat[c]), hr[c].get(hat[c]), drr[c].get(before[c]), dxr[c].get(dx);
#pragma unroll
                for (int j = 0; j < VEC; ++j) w[j] = gate[j] = q[c][j] = 0.f;
                if (at < g.d) factors_at(g.gamma, at, w), factors_at(g.post_gamma, at, q[c]), factors_at(g.gate, group * g.d + at, gate);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    q[c][j] *= g.b * gate[j];
                    hat[c][j] *= e;
                    rhat[c][j] = g.h ? s * fmaf(g.a, rhat[c][j], q[c][j] * hat[c][j]) : s * rhat[c][j];
                    const float t = dx[j] * w[j];
                    before[c][j] = fmaf(s, t, before[c][j]);
                    dgamma[c][j] = fmaf(dx[j], rhat[c][j], dgamma[c][j]);
                    const float qh = q[c][j] * hat[c][j];
                    sum[0] = fmaf(t, rhat[c][j], sum[0]), sum[1] = fmaf(qh, before[c][j], sum[1]), sum[2] = fmaf(qh, rhat[c][j], sum[2]);
                }
            }
            team_sum(sum);
            const float k = g.gamma.p ? s * sum[0] * per : 0.f, m = g.post_gamma.p ? (sum[1] - k * sum[2]) * per : 0.f;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int64_t at = (c * int(blockDim.x) + int(threadIdx.x)) * VEC, p = row * g.d + at;
                if (at >= g.d) break;
                float f[VEC], gate[VEC], out[VEC];
                factors_at(g.post_gamma, at, f), factors_at(g.gate, group * g.d + at, gate);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float D = fmaf(-k, rhat[c][j], before[c][j]);
                    out[j] = g.a * D;
                    const float bD = g.b * D;
                    dpost[c][j] = fmaf(gate[j] * bD, hat[c][j], dpost[c][j]);
                    dgate[c][j] = fmaf(f[j] * bD, hat[c][j], dgate[c][j]);
                    q[c][j] = e * fmaf(q[c][j], D, -hat[c][j] * m);
                }
                if (g.dr) put(g.dr + p, out);
                if (g.dh) put(g.dh + p, q[c]);
            }
        }
        if (g.gate.p) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int64_t at = (c * int(blockDim.x) + int(threadIdx.x)) * VEC;
                if (at >= g.d) break;
                if (g.pieces > 1) put(g.part_gate + unit * g.d + at, dgate[c]);
                else if (g.gate.bf16) put(static_cast<__nv_bfloat16*>(g.dgate) + group * g.d + at, dgate[c]);
                else put(static_cast<float*>(g.dgate) + group * g.d + at, dgate[c]);
            }
        }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int64_t at = (c * int(blockDim.x) + int(threadIdx.x)) * VEC;
        if (at >= g.d) break;
        if (g.part_gamma) put(g.part_gamma + team * g.d + at, dgamma[c]);
        if (g.part_post) put(g.part_post + team * g.d + at, dpost[c]);
    }
}

// out[group, c] = the sum of `count` rows of partial sums; 32 columns and 32 runs of rows a block
struct Join {
    const float* part;
    void* out;
    int64_t groups, count;
    int bf16;
};
struct Joins {
    Join j[3];
};
__global__ void __launch_bounds__(1024) join_kernel(const __grid_constant__ Joins all, int64_t d) {
    __shared__ float sums[32][33];
    after_previous();
    const Join& j   = all.j[blockIdx.z];
    const int64_t c = int64_t(blockIdx.x) * 32 + threadIdx.x;
    for (int64_t group = blockIdx.y; group < j.groups; group += gridDim.y) {
        const float* p = j.part + group * j.count * d + c;
        float v        = 0.f;
        if (c < d)
#pragma unroll 8
            for (int64_t k = threadIdx.y; k < j.count; k += 32) v += p[k * d];
        __syncthreads();
        sums[threadIdx.y][threadIdx.x] = v;
        __syncthreads();
        v                = warp_sum(sums[threadIdx.x][threadIdx.y]);  // a warp for each column
        const int64_t to = int64_t(blockIdx.x) * 32 + threadIdx.y;
        if (threadIdx.x == 0 && to < d) {
            if (j.bf16) static_cast<__nv_bfloat16*>(j.out)[group * d + to] = __float2bfloat16(v);
            else static_cast<float*>(j.out)[group * d + to] = v;
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
using Desc = mimk_residual_rmsnorm_desc;

bool float_type(int t) { return t == MIMK_F32 || t == MIMK_BF16; }
int check(const Desc* d) {
    if (!d || d->n < 0 || d->d < 0 || (d->gate && d->gate_rows < 1)) return MIMK_E_ARG;
    if (!float_type(d->stream_dtype) || !float_type(d->block_dtype) || (d->stream_dtype == MIMK_BF16 && d->block_dtype == MIMK_F32)) return MIMK_E_DTYPE;
    if ((d->gamma && !float_type(d->gamma_dtype)) || (d->post_gamma && !float_type(d->post_gamma_dtype)) || (d->gate && !float_type(d->gate_dtype))) return MIMK_E_DTYPE;
    if (!(d->eps >= 0)) return MIMK_E_ARG;
    if (d->n >= LIM || d->d > MOST_COLUMNS) return MIMK_E_UNSUPPORTED;
    if (!d->n || !d->d) return MIMK_OK;  // (operands without values have no address)
    if (!d->h && (d->post_gamma || d->gate || d->residual_scale != 1.f || d->branch_scale != 1.f)) return MIMK_E_ARG;
    if (!d->h && !d->gamma) return MIMK_E_ARG;  // (nothing to do)
    return MIMK_OK;
}
bool off(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % dtype_size(dtype) != 0; }
int misplaced(const Desc& d) {
    for (const void* p : {d.r, static_cast<const void*>(d.r_out), d.dr_out, static_cast<const void*>(d.dr)})
        if (off(p, d.stream_dtype)) return MIMK_E_ALIGN;
    for (const void* p : {d.h, static_cast<const void*>(d.x), d.dx, static_cast<const void*>(d.dh)})
        if (off(p, d.block_dtype)) return MIMK_E_ALIGN;
    if (off(d.gamma, d.gamma_dtype) || off(d.dgamma, d.gamma_dtype) || off(d.post_gamma, d.post_gamma_dtype) || off(d.dpost_gamma, d.post_gamma_dtype)) return MIMK_E_ALIGN;
    if (off(d.gate, d.gate_dtype) || off(d.dgate, d.gate_dtype) || off(d.kept, MIMK_F32)) return MIMK_E_ALIGN;
    return MIMK_OK;
}
bool vectors(const Desc& d) {
    bool all = d.d % 8 == 0;
    for (const void* p : {d.r, d.h, d.gamma, d.post_gamma, d.gate, static_cast<const void*>(d.r_out), static_cast<const void*>(d.x), d.dr_out, d.dx, static_cast<const void*>(d.dr),
                          static_cast<const void*>(d.dh), static_cast<const void*>(d.dgate)})
        all = all && aligned16(p);
    return all;
}

// How rows are dealt out: threads and rows of a block, and for the backward pass blocks and units of rows.
struct Plan {
    int threads, rows, blocks;
    int64_t groups, pieces;
    float *gamma, *post, *gate;
};
Plan plan(const Desc& d, bool vec, Space& space, int sm_count) {
    Plan p{};
    const int64_t each = d.d <= 2048 ? 8 : d.d <= 8192 ? 16 : 32, lanes = up((d.d + each - 1) / each, 32);
    (void)vec;
    p.threads = int(lanes), p.rows = lanes == 32 ? 4 : 1;
    // (registers for 512 threads or so of 16 columns with their three sums on an SM)
    const int64_t most = int64_t(sm_count) * (lanes <= 128 ? 4 : lanes <= 256 ? 2 : 1), need = (d.n + p.rows - 1) / p.rows;
    p.blocks = int(need < most ? (need < 1 ? 1 : need) : most);
    const int64_t teams = int64_t(p.blocks) * p.rows, run = d.gate ? d.gate_rows : (d.n > 0 ? d.n : 1);
    p.groups = (d.n + run - 1) / run;
    p.pieces = p.groups ? (teams + p.groups - 1) / p.groups : 1;
    if (p.pieces > run) p.pieces = run;
    auto part = [&](int64_t rows) { return static_cast<float*>(space.take(size_t(rows) * size_t(d.d) * 4)); };
    if (d.gamma) p.gamma = part(teams);
    if (d.post_gamma) p.post = part(teams);
    if (d.gate && p.pieces > 1) p.gate = part(p.groups * p.pieces);
    return p;
}

template <class RT, class HT>
Args<RT, HT> args_of(const Desc& d) {
    Args<RT, HT> g{};
    g.n = d.n, g.d = d.d, g.gate_rows = d.gate ? d.gate_rows : (d.n > 0 ? d.n : 1);
    g.r = static_cast<const RT*>(d.r), g.h = static_cast<const HT*>(d.h);
    g.gamma = {d.gamma, d.gamma_dtype == MIMK_BF16}, g.post_gamma = {d.post_gamma, d.post_gamma_dtype == MIMK_BF16}, g.gate = {d.gate, d.gate_dtype == MIMK_BF16};
    g.r_out = static_cast<RT*>(d.r_out), g.x = static_cast<HT*>(d.x), g.kept = d.kept;
    g.dr_out = static_cast<const RT*>(d.dr_out), g.dx = static_cast<const HT*>(d.dx), g.dr = static_cast<RT*>(d.dr), g.dh = static_cast<HT*>(d.dh);
    g.dgate = d.dgate, g.eps = d.eps, g.a = d.residual_scale, g.b = d.branch_scale;
    return g;
}

template <class RT, class HT, int VEC>
int forward(const Desc& d, const Plan& p, const DeviceInfo& dev, cudaStream_t s) {
    const Args<RT, HT> g = args_of<RT, HT>(d);
    const auto kern = d.d <= 2048 ? forward_kernel<RT, HT, VEC, 8 / VEC, 256> : d.d <= 8192 ? forward_kernel<RT, HT, VEC, 16 / VEC, 512> : forward_kernel<RT, HT, VEC, 32 / VEC, 1024>;
    const int64_t blocks = (d.n + p.rows - 1) / p.rows;
    cudaLaunchAttribute early = {};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization, early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(unsigned(blocks < (1 << 20) ? blocks : 1 << 20)), config.blockDim = dim3(p.threads, p.rows), config.stream = s, config.attrs = &early, config.numAttrs = 1;
    return note_cuda_error(cudaLaunchKernelEx(&config, kern, g));
}
template <class RT, class HT, int VEC>
int backward(const Desc& d, const Plan& p, const DeviceInfo& dev, cudaStream_t s) {
    Args<RT, HT> g = args_of<RT, HT>(d);
    g.part_gamma = p.gamma, g.part_post = p.post, g.part_gate = p.gate, g.groups = p.groups, g.pieces = p.pieces;
    const auto kern = d.d <= 2048 ? backward_kernel<RT, HT, VEC, 8 / VEC, 256> : d.d <= 8192 ? backward_kernel<RT, HT, VEC, 16 / VEC, 512> : backward_kernel<RT, HT, VEC, 32 / VEC, 1024>;
    cudaLaunchAttribute early = {};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization, early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(unsigned(p.blocks)), config.blockDim = dim3(p.threads, p.rows), config.stream = s, config.attrs = &early, config.numAttrs = 1;
    MIMK_TRY(note_cuda_error(cudaLaunchKernelEx(&config, kern, g)));
    Joins all{};
    int count           = 0;
    int64_t most        = 1;
    const int64_t teams = int64_t(p.blocks) * p.rows;
    if (p.gamma) all.j[count++] = {p.gamma, d.dgamma, 1, teams, d.gamma_dtype == MIMK_BF16};
    if (p.post) all.j[count++] = {p.post, d.dpost_gamma, 1, teams, d.post_gamma_dtype == MIMK_BF16};
    if (p.gate) all.j[count++] = {p.gate, d.dgate, p.groups, p.pieces, d.gate_dtype == MIMK_BF16}, most = p.groups;
    if (!count) return MIMK_OK;
    config.gridDim = dim3(unsigned((d.d + 31) / 32), unsigned(most < 65535 ? most : 65535), unsigned(count)), config.blockDim = dim3(32, 32);
    return note_cuda_error(cudaLaunchKernelEx(&config, join_kernel, all, d.d));
}

#define MIMK_BY_TYPES(F, VEC, ...)                                                                        \
    (d->stream_dtype == MIMK_BF16  ? F<__nv_bfloat16, __nv_bfloat16, VEC>(__VA_ARGS__)                    \
     : d->block_dtype == MIMK_BF16 ? F<float, __nv_bfloat16, VEC>(__VA_ARGS__)                            \
                                   : F<float, float, VEC>(__VA_ARGS__))

int zero(void* p, int64_t count, int dtype, cudaStream_t s) {
    if (p && count) MIMK_CUDA_TRY(cudaMemsetAsync(p, 0, size_t(count) * dtype_size(dtype), s));
    return MIMK_OK;
}

}  // namespace
}  // namespace mimk

using namespace mimk;

extern "C" int mimk_residual_rmsnorm_fwd(const mimk_residual_rmsnorm_desc* d, void* stream) {
    MIMK_TRY(check(d));
    int st                = MIMK_OK;
    const DeviceInfo* dev = device_info(&st);
    if (!dev) return st;
    if (!d->n || !d->d) return MIMK_OK;
    if (!d->r || (d->gamma && !d->x) || (d->h && !d->r_out) || (!d->h && d->r_out) || (!d->gamma && d->x)) return MIMK_E_ARG;
    MIMK_TRY(misplaced(*d));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    Space space(nullptr);
    const bool vec = vectors(*d);
    const Plan p   = plan(*d, vec, space, dev->sm_count);
    return vec ? MIMK_BY_TYPES(forward, 8, *d, p, *dev, s) : MIMK_BY_TYPES(forward, 1, *d, p, *dev, s);
}

extern "C" int mimk_residual_rmsnorm_workspace(const mimk_residual_rmsnorm_desc* d, uint64_t* bytes) {
    MIMK_TRY(check(d));
    if (!bytes) return MIMK_E_ARG;
    int st                = MIMK_OK;
    const DeviceInfo* dev = device_info(&st);
    if (!dev) return st;
    Space space(nullptr);
    plan(*d, false, space, dev->sm_count);
    *bytes = space.used();
    return MIMK_OK;
}

extern "C" int mimk_residual_rmsnorm_bwd(const mimk_residual_rmsnorm_desc* d, void* stream) {
    MIMK_TRY(check(d));
    int st                = MIMK_OK;
    const DeviceInfo* dev = device_info(&st);
    if (!dev) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (!d->d) return MIMK_OK;
    if ((d->gamma && !d->dgamma) || (d->post_gamma && !d->dpost_gamma)) return MIMK_E_ARG;
    if (!d->n) {  // (dgate has no rows)
        MIMK_TRY(zero(d->dgamma, d->gamma ? d->d : 0, d->gamma_dtype, s));
        return zero(d->dpost_gamma, d->post_gamma ? d->d : 0, d->post_gamma_dtype, s);
    }
    if (!d->r || !d->dr || (d->h && !d->dh) || (!d->h && d->dh) || (d->gate && !d->dgate) || (d->gamma ? !d->dx : d->dx != nullptr)) return MIMK_E_ARG;
    if ((d->gamma || d->post_gamma) && !d->kept) return MIMK_E_ARG;
    MIMK_TRY(misplaced(*d));
    Space space(d->workspace);
    const bool vec = vectors(*d);
    const Plan p   = plan(*d, vec, space, dev->sm_count);
    if (space.used() > d->workspace_bytes || (space.used() && !d->workspace)) return MIMK_E_WORKSPACE;
    if (space.used() && !aligned16(d->workspace)) return MIMK_E_ALIGN;
    return vec ? MIMK_BY_TYPES(backward, 8, *d, p, *dev, s) : MIMK_BY_TYPES(backward, 1, *d, p, *dev, s);
}
