// Softmax cross-entropy of a linear layer, l = x W over a large number of classes, without the logits: loss, and the gradients of x and W.
//
//   lse_i = log sum_j exp(l_ij),  loss_i = lse_i - l_i,t(i)
//   p_ij = g_i (exp(l_ij - lse_i) - [j = t(i)]),  dx = p W^T,  dW = x^T p        g: the loss's gradient, over the count for a mean
//
// bf16: the logits exist as accumulators only. A first product reduces each 128 columns of a row to a maximum and a sum of exponentials
// (8 bytes for 128 logits); a kernel over rows joins them: 8192 x 4096 x 131072 in 6.7 to 7.0 ms. Loss and gradients in one call: where n v
// is at most 2^30, that product also leaves the exponentials themselves in 16 bits (ten of them significant, where p has eight: as bf16
// they would round p twice), which a pass over them turns into p once the sums are known (the targets' p from their logits, in f32), and
// one launch makes dW and dx: 6 n d v operations. Beyond that, and for gradients from an earlier call's lse, by pieces of the classes: a
// product writes p of the piece as bf16, and one launch makes the piece's rows of dW and adds to dx in f32, with the logits over again in the one
// call: 8 n d v operations, and 512 MiB of p. 8192 rows of that size at once: 24.7 to 26.0 ms at the power limit (1.02 to 1.07 PFLOP/s of
// the 6 n d v; library products of 8192^3 there: 1.36), 21.5 to 23.4 in a short run; by pieces 26.1 to 27.5 in such a run, the gradients
// alone 20.2 to 21.4. 2^30 is a limit of memory (2 GiB of exponentials): 8193 rows take 27.3 to 28.6 by pieces and would take 22.2 to 23.4
// without it, 16384 rows 52.8 to 54.2 and 49.6 to 52.3 (4 GiB).
// f32: pieces of rows instead, through the library's f32 products, with the logits of a piece in memory, turned into p in place. 512 x 784 x
// 10007: 398 us, the loss alone 150, the gradients alone 385; 361 of the 398 are the products, whose faster kernel wants rows of whole 16 bytes.
//
// Rows without a target (the ignored index) are taken out first: the rows that are left are copied together, and the products run over as
// many rows as a count in device memory says. What the other rows hold, NaN included, is never read.
#include <algorithm>

#include "train_common.cuh"

namespace mimk {

namespace {

using namespace group;

constexpr int64_t LIM = int64_t(1) << 30;
constexpr int64_t PIECE_CELLS = int64_t(1) << 28;  // bf16: p of a piece, 512 MiB
constexpr int64_t KEPT_CELLS  = int64_t(1) << 30;  // bf16: exponentials that are kept until the sums are known, 2 GiB
constexpr int64_t PIECE_FLOATS = int64_t(1) << 27; // f32: logits of a piece, 512 MiB

struct Rows {             // per row that is left (all of them without an ignored index)
    int* target;          // its column, or -1: none that exists
    int* index;           // its place in x; null: the same
    int* place;           // [n] the other way round, -1 for a row that was taken out; null: the same
    int* count;           // rows that are left; rows with a target that exists; CTAs that have finished
    float *lse, *scale;   // log of the sum; what the row's part of the gradient is multiplied by
    float* loss;          // [n], by place in x
    float* target_logit;
    float2* part;
};

// ---- rows ------------------------------------------------------------------------------------------------------------------------
// One CTA: every thread counts the rows that are left among its share, then writes them behind those of the threads before it.
template <class I>
__global__ void __launch_bounds__(1024) prepare_kernel(const I* __restrict__ targets, int64_t n, int64_t v, bool has_ignore, int64_t ignore, Rows r,
                                                      float* lse_out, int* status) {
    __shared__ int warp_total[32], warp_exist[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t per = (n + 1023) / 1024;
    const int64_t from = threadIdx.x * per < n ? threadIdx.x * per : n, to = from + per < n ? from + per : n;
    // (the ignored index may be a class, as a padding token's is)
    const auto has_target = [&](int64_t t) { return t >= 0 && t < v && !(has_ignore && t == ignore); };
    int mine = 0, exist = 0;
    for (int64_t i = from; i < to; ++i) {
        const int64_t t  = targets[i];
        const bool there = has_target(t);
        exist += there, mine += r.index ? there : 1;
    }
    int before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, before, o);
        before += lane >= o ? x : 0;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) exist += __shfl_xor_sync(0xffffffffu, exist, o);
    if (lane == 31) warp_total[warp] = before, warp_exist[warp] = exist;
    __syncthreads();
    int at = before - mine, all = 0;
    exist = 0;
    for (int w = 0; w < 32; ++w) {
        at += w < warp ? warp_total[w] : 0;
        all += warp_total[w], exist += warp_exist[w];
    }
    if (threadIdx.x == 0) r.count[0] = all, r.count[1] = exist, r.count[2] = 0;
    for (int64_t i = from; i < to; ++i) {
        const int64_t t  = targets[i];
        const bool there = has_target(t), ignored = has_ignore && t == ignore;
        if (!there && !ignored) *status = MIMK_E_SHAPE;
        if (!r.index) {
            r.target[i] = there ? int(t) : -1;
        } else if (there) {
            r.target[at] = int(t), r.index[at] = int(i), r.place[i] = at++;
        } else {
            r.place[i] = -1;
            if (r.loss) r.loss[i] = ignored ? 0.f : __int_as_float(0x7fc00000);
            if (lse_out) lse_out[i] = 0.f;
        }
    }
}

// The rows that are left, together; zeros up to the end of the last 64 of them (all of them for f32 products, which know no count).
template <class V>
__global__ void gather_rows_kernel(const V* __restrict__ x, int64_t cols, int64_t from_pitch, V* __restrict__ to, int64_t to_pitch, const int* __restrict__ index,
                                   const int* __restrict__ count, int64_t n, bool all) {
    const int64_t left = *count, end = all ? n : (left + 63) / 64 * 64 < n ? (left + 63) / 64 * 64 : n;
    for (int64_t r = blockIdx.x; r < end; r += gridDim.x) {
        const int64_t from = r < left ? (index ? index[r] : r) : -1;
        for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) to[r * to_pitch + c] = from >= 0 ? x[from * from_pitch + c] : V{};
    }
}

__device__ __forceinline__ float scale_of(const Rows& r, int64_t row, int target, const float* dloss, int reduction) {
    if (target < 0) return 0.f;
    const float g = dloss ? dloss[reduction == MIMK_REDUCTION_NONE ? row : 0] : 1.f;
    return reduction == MIMK_REDUCTION_MEAN ? g / float(max(r.count[1], 1)) : g;
}
// the sum of all rows' losses by the last CTA to come here, always in the same order
__device__ void finish_loss(const Rows& r, int64_t n, int reduction, float* loss) {
    __shared__ bool last;
    __shared__ double part[32];
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(r.count + 2, 1) == int(gridDim.x) - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    double sum = 0;
    for (int64_t i = threadIdx.x; i < n; i += blockDim.x) sum += double(__ldcg(r.loss + i));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (unsigned w = 1; w < blockDim.x / 32; ++w) sum += part[w];
        *loss = float(reduction == MIMK_REDUCTION_MEAN ? sum / max(r.count[1], 1) : sum);
    }
}

// The maxima and sums of a row's parts joined, a CTA for a row: the largest maximum first, then the sums scaled to it, so that no load waits for another's
// exponential (one pass by a warp took 14 us for the 1024 parts of one row). loss: the reduced one, or null.
__global__ void __launch_bounds__(128) join_kernel(Rows r, int64_t n, int parts, const float* dloss, int reduction, float* loss, float* lse_out) {
    after_previous();
    __shared__ float warp_top[4], warp_sums[4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int left = r.count[0];
    for (int64_t j = blockIdx.x; j < left; j += gridDim.x) {
        const float2* part = r.part + j * parts;
        float top = -INFINITY, sum = 0.f;
#pragma unroll 8
        for (int t = threadIdx.x; t < parts; t += 128) top = fmaxf(top, part[t].x);
        top = warp_max(top);
        if (lane == 0) warp_top[warp] = top;
        __syncthreads();
        top = fmaxf(fmaxf(warp_top[0], warp_top[1]), fmaxf(warp_top[2], warp_top[3]));
#pragma unroll 8
        for (int t = threadIdx.x; t < parts; t += 128) {
            const float2 p = part[t];
            sum += p.x == -INFINITY ? p.y : p.y * __expf(p.x - top);  // (a maximum of -inf has a sum of zero, or NaN)
        }
        sum = warp_sum(sum);
        if (lane == 0) warp_sums[warp] = sum;
        __syncthreads();
        if (threadIdx.x == 0) {
            const int64_t row = r.index ? r.index[j] : j;
            const int target  = r.target[j];
            const float lse   = top + logf((warp_sums[0] + warp_sums[1]) + (warp_sums[2] + warp_sums[3]));
            r.lse[j]          = lse;
            if (r.scale) r.scale[j] = scale_of(r, row, target, dloss, reduction);
            if (lse_out) lse_out[row] = lse;
            if (r.loss) r.loss[row] = target < 0 ? __int_as_float(0x7fc00000) : lse - r.target_logit[j];
        }
    }
    if (loss) finish_loss(r, n, reduction, loss);
}

// ---- a few rows ------------------------------------------------------------------------------------------------------------------
// The forward pass of up to FEW rows with W stored [v, d]: its bytes bound it, and a tile of 256 rows keeps half of shared memory for zeros. A warp takes
// four classes at a time, a lane 16 bytes of each; the rows of x are in shared memory as f32, split in halves of eight values so that neighbouring
// lanes read neighbouring 16 bytes. Calls of 1, 2, 3, 4 rows of 4096 against 131072 classes: 169, 185, 211, 210 to 218 us (one row: 6.5 TB/s), by the
// tensor cores' pass 269, 224, 231, 252. Two rows have a kernel of their own (as two of four: 204), with 92 bytes of spills in its 64 registers.
// Five rows would be two rounds of this kernel; the tensor cores take 245, and 195 for 16 or 32.
// GRAD: gradients from the lse of such a pass take their logits from here, too, to the same bits (those of the tensor cores are 2e-6 of themselves off at
// 1024 features, which 1 - p of a row that is nearly certain does not bear): p of the `n` rows, zeros for those that were taken out. Gradients of
// 1, 2, 4 rows: 650, 672, 695 us; with p from the tensor cores 730 to 800.
constexpr int FEW = 4, FEW_CTAS = 4;
template <int N, bool GRAD>
__global__ void __launch_bounds__(256, N == FEW ? 2 : FEW_CTAS) few_rows_kernel(const __nv_bfloat16* x, int64_t x_pitch, const __nv_bfloat16* w, int d, int v,
                                                                  Rows r, int n, int column0, __nv_bfloat16* p, int64_t pitch) {
    after_previous();
    extern __shared__ float4 xs[];  // [N][2][d / 8]
    const int lane = threadIdx.x & 31, eighths = d / 8, slots = gridDim.x * 8, slot = blockIdx.x * 8 + (threadIdx.x >> 5);
    const int left = r.count[0];
    for (int i = threadIdx.x; i < N * eighths; i += 256) {
        const int j = i / eighths, k = i - j * eighths;
        uint4 u     = make_uint4(0, 0, 0, 0);
        if (j < left) u = *reinterpret_cast<const uint4*>(x + int64_t(r.index ? r.index[j] : j) * x_pitch + k * 8);
        xs[j * 2 * eighths + k] = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
        xs[(j * 2 + 1) * eighths + k] =
            make_float4(__uint_as_float(u.z << 16), __uint_as_float(u.z & 0xffff0000u), __uint_as_float(u.w << 16), __uint_as_float(u.w & 0xffff0000u));
    }
    __syncthreads();
    const bool mine  = lane < N && lane < left;  // lane j looks after row j
    const int target = mine ? r.target[lane] - column0 : -1;
    const float lse = GRAD && mine ? r.lse[lane] : 0.f, scale = GRAD && mine ? r.scale[lane] : 0.f;
    float top = -INFINITY, sum = 0.f;
    for (int64_t c = int64_t(slot) * 4; c < v; c += int64_t(slots) * 4) {
        float acc[4][N];
        const uint4* at[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            at[i] = reinterpret_cast<const uint4*>(w + (c + i < v ? c + i : v - 1) * int64_t(d));
#pragma unroll
            for (int j = 0; j < N; ++j) acc[i][j] = 0.f;
        }
#pragma unroll 2
        for (int k = lane; k < eighths; k += 32) {
            uint4 u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = __ldcs(at[i] + k);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float4 a = xs[j * 2 * eighths + k], b = xs[(j * 2 + 1) * eighths + k];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    acc[i][j] = fmaf(__uint_as_float(u[i].x << 16), a.x, fmaf(__uint_as_float(u[i].x & 0xffff0000u), a.y, acc[i][j]));
                    acc[i][j] = fmaf(__uint_as_float(u[i].y << 16), a.z, fmaf(__uint_as_float(u[i].y & 0xffff0000u), a.w, acc[i][j]));
                    acc[i][j] = fmaf(__uint_as_float(u[i].z << 16), b.x, fmaf(__uint_as_float(u[i].z & 0xffff0000u), b.y, acc[i][j]));
                    acc[i][j] = fmaf(__uint_as_float(u[i].w << 16), b.z, fmaf(__uint_as_float(u[i].w & 0xffff0000u), b.w, acc[i][j]));
                }
            }
        }
        float l[4] = {};
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float all = warp_sum(acc[i][j]);
                l[i]            = lane == j ? all : l[i];
            }
        if constexpr (GRAD) {
#pragma unroll
            for (int i = 0; i < 4; ++i) l[i] = mine && c + i < v ? scale * (__expf(l[i] - lse) - (target == c + i ? 1.f : 0.f)) : 0.f;
            // (rows of p are of whole 256 columns)
            if (lane < n) *reinterpret_cast<uint2*>(p + lane * pitch + c) = make_uint2(pack_bf16x2(l[0], l[1]), pack_bf16x2(l[2], l[3]));
        } else if (lane < N) {
            float most = top;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (c + i >= v) l[i] = -INFINITY;
                else if (target == c + i) r.target_logit[lane] = l[i];
                most = fmaxf(most, l[i]);
            }
            if (most > top) sum *= top == -INFINITY ? 1.f : __expf(top - most), top = most;  // (an earlier sum at -inf is zero, or NaN)
            const float base = top == -INFINITY ? 0.f : top;
            sum += (__expf(l[0] - base) + __expf(l[1] - base)) + (__expf(l[2] - base) + __expf(l[3] - base));
        }
    }
    if (!GRAD && mine) r.part[int64_t(lane) * slots + slot] = make_float2(top, sum);
}

// p from the exponentials, in place: exp(l - m) becomes scale exp(l - lse) as bf16, less scale at the target, whose own value comes from its
// logit; zeros in the rows up to the end of the last 64, which the products over rows read. A warp takes 1024 columns of a row, a lane four times 16
// bytes. Bound by the bytes: 0.78 ms for
// 8192 x 131072, 5.5 TB/s.
__global__ void __launch_bounds__(256) probabilities_kernel(Rows r, uint16_t* __restrict__ p, int64_t pitch, int64_t n, int parts) {
    after_previous();
    const int lane = threadIdx.x & 31;
    const int left = r.count[0];
    const int64_t end = min(n, (int64_t(left) + 63) / 64 * 64);
    const int first   = (int(blockIdx.x) * 8 + int(threadIdx.x >> 5)) * 1024 + lane * 8;
    for (int64_t j = blockIdx.y; j < end; j += gridDim.y) {
        const bool there = j < left;
        const float lse  = there ? r.lse[j] : 0.f, scale = there ? r.scale[j] : 0.f;
        const int target = there ? r.target[j] : -1;
        uint4 v[4];
        float top[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = first + i * 256;
            if (c >= pitch) continue;
            v[i]   = there ? *reinterpret_cast<const uint4*>(p + j * pitch + c) : make_uint4(0, 0, 0, 0);
            top[i] = there ? r.part[j * parts + (c >> 7)].x : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = first + i * 256;
            if (c >= pitch) continue;
            const float by = scale * __expf(top[i] - lse);
            uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float lo = exp_of(w[e] & 0xffffu) * by, hi = exp_of(w[e] >> 16) * by;
                if (target - c == 2 * e) lo = scale * (__expf(r.target_logit[j] - lse) - 1.f);
                if (target - c == 2 * e + 1) hi = scale * (__expf(r.target_logit[j] - lse) - 1.f);
                w[e] = there ? pack_bf16x2(lo, hi) : 0u;
            }
            *reinterpret_cast<uint4*>(p + j * pitch + c) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// the rows' logarithms from an earlier call, and their scales
__global__ void recall_kernel(Rows r, const float* __restrict__ lse, const float* dloss, int reduction) {
    const int left = r.count[0];
    for (int64_t j = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; j < left; j += int64_t(gridDim.x) * blockDim.x) {
        const int64_t row = r.index ? r.index[j] : j;
        r.lse[j]          = lse[row];
        r.scale[j]        = scale_of(r, row, r.target[j], dloss, reduction);
    }
}

// dx from its partial sums, each row to its place; zeros for the rows that were taken out. Four columns a thread.
template <class T>
__global__ void place_rows_kernel(const float* part, int splits, int64_t stride, int64_t pitch, const int* place, T* dx,
                                  int64_t n, int64_t cols, bool words) {
    after_previous();
    const int64_t quads = (cols + 3) / 4, all = n * quads;
    for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < all; i += int64_t(gridDim.x) * blockDim.x) {
        const int64_t row = i / quads, c = (i - row * quads) * 4, j = place ? place[row] : row;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (j >= 0) {
            for (int s = 0; s < splits; ++s) {
                const float* at = part + s * stride + j * pitch + c;
                if (pitch % 4 == 0) {
                    const float4 w = *reinterpret_cast<const float4*>(at);
                    v[0] += w.x, v[1] += w.y, v[2] += w.z, v[3] += w.w;
                } else {
                    for (int e = 0; e < 4 && c + e < cols; ++e) v[e] += at[e];
                }
            }
        }
        T* o = dx + row * cols + c;
        if (sizeof(T) == 2 && words && c + 4 <= cols) {
            *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
        } else {
            for (int e = 0; e < 4 && c + e < cols; ++e) o[e] = T(v[e]);
        }
    }
}

// ---- f32: rows of logits in memory -------------------------------------------------------------------------------------------------
// A CTA per row of a piece that starts at row `first`: log of the sum and loss, or the logarithm of an earlier call (`earlier`, by place in x), and the row
// turned into p where the gradient is wanted.
__global__ void __launch_bounds__(512) logits_kernel(float* __restrict__ logits, int64_t v, int64_t first, Rows r, const float* dloss, int reduction,
                                                     const float* earlier, float* lse_out, bool grad) {
    __shared__ float warp_top[16], warp_part[16];
    const int64_t j = first + blockIdx.x;
    float* row      = logits + int64_t(blockIdx.x) * v;
    if (j >= r.count[0]) {
        if (grad)
            for (int64_t c = threadIdx.x; c < v; c += blockDim.x) row[c] = 0.f;
        return;
    }
    const int target    = r.target[j];
    const int64_t place = r.index ? r.index[j] : j;
    // p = exp(l - base) over
    float base = 0.f, over = 1.f;
    if (earlier) {
        base = earlier[place];
    } else {
        float top = -INFINITY, sum = 0.f;
        for (int64_t c = threadIdx.x; c < v; c += blockDim.x) top = fmaxf(top, row[c]);
        top = warp_max(top);
        if ((threadIdx.x & 31) == 0) warp_top[threadIdx.x >> 5] = top;
        __syncthreads();
        for (unsigned w = 0; w < blockDim.x / 32; ++w) top = fmaxf(top, warp_top[w]);
        for (int64_t c = threadIdx.x; c < v; c += blockDim.x) sum += expf(row[c] - top);
        sum = warp_sum(sum);
        if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x >> 5] = sum;
        const float at = target >= 0 ? row[target] : 0.f;
        __syncthreads();  // (every thread has the target's logit before the row changes)
        sum = 0.f;
        for (unsigned w = 0; w < blockDim.x / 32; ++w) sum += warp_part[w];
        if (threadIdx.x == 0) {
            const float lse = top + logf(sum);
            if (lse_out) lse_out[place] = lse;
            if (r.loss) r.loss[place] = target < 0 ? __int_as_float(0x7fc00000) : lse - at;
        }
        base = top, over = 1.f / sum;
    }
    if (grad) {
        const float scale = scale_of(r, place, target, dloss, reduction);
        for (int64_t c = threadIdx.x; c < v; c += blockDim.x) {
            const float p = expf(row[c] - base) * over;
            row[c]        = scale * (c == target ? p - 1.f : p);
        }
    }
}
__global__ void loss_kernel(Rows r, int64_t n, int reduction, float* loss) { finish_loss(r, n, reduction, loss); }

__global__ void add_kernel(float* __restrict__ to, const float* __restrict__ from, int64_t n) {
    for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < n; i += int64_t(gridDim.x) * blockDim.x) to[i] += from[i];
}

unsigned grid_for(int64_t items, int per, int64_t most) {
    const int64_t blocks = (items + per - 1) / per;
    return unsigned(blocks < 1 ? 1 : blocks < most ? blocks : most);
}

// ---- plan ------------------------------------------------------------------------------------------------------------------------
struct Plan {
    Rows rows{};
    void* x;  // the rows that are left, together, or null: the caller's
    int64_t x_pitch;
    Staged w, dw;
    int parts;                  // of a row, whose maxima and sums are joined
    bool few;
    int64_t piece;              // columns (bf16) or rows (f32) of a piece
    bool kept;                  // bf16: the forward product leaves its exponentials, and all columns are one piece
    void* p;                    // bf16: p of a piece; f32: its logits
    float* dx;                  // partial sums of dx (bf16), or dx of the rows that are left (f32)
    int splits;
    int64_t rows_pad, dx_pitch;
    void *turned, *sum;         // f32: x or p transposed; a piece's part of dW
    void* cut;                  // f32: operands that a product cuts beforehand, or null
};

// One product of the f32 form.
mimk_gemm_desc product(int64_t m, int64_t n, int64_t k, const void* a, const void* b, int layout, void* c) {
    mimk_gemm_desc g = {};
    g.batch = 1, g.m = m, g.n = n, g.k = k, g.a = a, g.b = b, g.c = c;
    g.in_dtype = g.out_dtype = MIMK_F32, g.b_layout = layout;
    return g;
}
// What the products of a piece of `rows` rows need for their operands.
size_t cut_bytes(const mimk_linear_ce_desc& d, int64_t rows, bool backward, int sm_count) {
    const bool nk     = d.w_layout == MIMK_B_NK;
    const auto needed = [&](int64_t m, int64_t n, int64_t k, int layout) { return gemm_f32_scratch(product(m, n, k, nullptr, nullptr, layout, nullptr), sm_count); };
    if (!rows) return 0;
    size_t bytes = needed(rows, d.v, d.d, d.w_layout);
    if (backward) {
        bytes = std::max(bytes, needed(rows, d.d, d.v, nk ? MIMK_B_KN : MIMK_B_NK));
        bytes = std::max(bytes, nk ? needed(d.v, d.d, rows, MIMK_B_KN) : needed(d.d, d.v, rows, MIMK_B_KN));
    }
    return bytes;
}

Plan plan(const mimk_linear_ce_desc& d, bool forward, bool backward, Space& space, int sm_count) {
    Plan p{};
    const size_t n = size_t(d.n);
    auto ints      = [&](size_t k) { return static_cast<int*>(space.take(k * 4)); };
    auto floats    = [&](size_t k) { return static_cast<float*>(space.take(k * 4)); };
    const bool taken = d.has_ignore != 0;
    p.rows.target = ints(n), p.rows.count = ints(4);
    if (taken) p.rows.index = ints(n), p.rows.place = ints(n);
    p.rows.lse = floats(n);
    if (backward) p.rows.scale = floats(n);
    if (forward) p.rows.loss = d.reduction == MIMK_REDUCTION_NONE ? d.loss : floats(n);
    if (d.dtype == MIMK_F32) {
        p.x_pitch = d.d;
        if (taken) p.x = space.take(n * size_t(d.d) * 4);
        p.piece = std::max<int64_t>(1, std::min(d.n, PIECE_FLOATS / d.v));
        p.p     = space.take(size_t(p.piece) * size_t(d.v) * 4);
        if (backward) {
            const bool nk = d.w_layout == MIMK_B_NK;
            if (taken) p.dx = floats(n * size_t(d.d));
            p.turned = space.take(size_t(p.piece) * size_t(nk ? d.v : d.d) * 4);
            if (p.piece < d.n) p.sum = space.take(size_t(d.d) * size_t(d.v) * 4);
        }
        const size_t cut = std::max(cut_bytes(d, p.piece, backward, sm_count), cut_bytes(d, d.n % p.piece, backward, sm_count));
        if (cut) p.cut = space.take(cut);
        return p;
    }
    p.x_pitch = d.d;
    if (taken || !tma_can_read(d.x, d.d)) p.x_pitch = up(d.d, 8), p.x = space.take(n * size_t(p.x_pitch) * 2);
    const bool nk = d.w_layout == MIMK_B_NK;
    p.w           = nk ? stage(space, d.w, d.v, d.d) : stage(space, d.w, d.d, d.v);
    // (up to 64 KiB of shared memory: FEW_CTAS CTAs to an SM; loss and gradients at once: the tensor cores' pass leaves the exponentials, too)
    p.few   = forward != backward && nk && d.n <= FEW && (d.n <= 2 ? d.n : FEW) * d.d <= 16384 && !p.w.copied() && tma_can_read(d.x, d.d);
    p.parts = p.few ? sm_count * FEW_CTAS * 8 : int((d.v + 255) / 256) * 2;
    if (p.few && forward) p.x = nullptr;
    if (forward) p.rows.part = static_cast<float2*>(space.take(n * size_t(p.parts) * 8)), p.rows.target_logit = floats(n);
    if (backward) {
        p.dw    = nk ? stage(space, d.dw, d.v, d.d) : stage(space, d.dw, d.d, d.v);
        p.kept  = forward && d.n * up(d.v, 8) <= KEPT_CELLS;
        p.piece = p.kept ? up(d.v, 8) : std::min(up(d.v, 256), std::max<int64_t>(4096, PIECE_CELLS / d.n / 256 * 256));
        p.p     = space.take(n * size_t(p.piece) * 2);
        p.splits   = pick_splits(d.n, d.d, std::min(d.v, p.piece) / 64 + 1, sm_count);
        p.rows_pad = up(d.n, 32), p.dx_pitch = up(d.d, 4);
        // (a sum of several pieces is kept in f32, and so is one whose rows go elsewhere or whose matrix TMA cannot write)
        if (p.splits > 1 || p.piece < d.v || taken || !tma_can_read(d.dx, d.d)) p.dx = floats(size_t(p.splits) * size_t(p.rows_pad) * size_t(p.dx_pitch));
    }
    return p;
}

int check(const mimk_linear_ce_desc* d) {
    if (!d) return MIMK_E_ARG;
    if (d->n < 0 || d->d < 0 || d->v < 0) return MIMK_E_ARG;
    if (d->dtype != MIMK_BF16 && d->dtype != MIMK_F32) return MIMK_E_DTYPE;
    if (d->target_dtype != MIMK_I32 && d->target_dtype != MIMK_I64) return MIMK_E_DTYPE;
    if (d->w_layout != MIMK_B_KN && d->w_layout != MIMK_B_NK) return MIMK_E_ARG;
    if (d->reduction < MIMK_REDUCTION_NONE || d->reduction > MIMK_REDUCTION_SUM) return MIMK_E_ARG;
    if (d->n >= LIM || d->d >= LIM || d->v >= LIM) return MIMK_E_UNSUPPORTED;
    // a class there is no score for: with rows there has to be a class, and with classes a feature
    if (d->n > 0 && (d->v == 0 || d->d == 0)) return MIMK_E_SHAPE;
    return MIMK_OK;
}

// The rows that are left, and x of them.
int begin(const mimk_linear_ce_desc& d, const Plan& p, bool forward, const DeviceInfo& dev, cudaStream_t s) {
    float* lse_out = forward ? d.lse : nullptr;
    if (d.target_dtype == MIMK_I64)
        prepare_kernel<int64_t><<<1, 1024, 0, s>>>(static_cast<const int64_t*>(d.targets), d.n, d.v, d.has_ignore != 0, d.ignore_index, p.rows, lse_out, dev.status_dev);
    else
        prepare_kernel<int32_t><<<1, 1024, 0, s>>>(static_cast<const int32_t*>(d.targets), d.n, d.v, d.has_ignore != 0, d.ignore_index, p.rows, lse_out, dev.status_dev);
    MIMK_TRY(launch_status());
    if (!p.x) return MIMK_OK;
    const unsigned grid = grid_for(d.n, 1, 65535);
    const int size      = d.dtype == MIMK_BF16 ? 2 : 4;
    const bool all      = d.dtype == MIMK_F32;
    if (aligned16(d.x) && d.d * size % 16 == 0)
        gather_rows_kernel<uint4><<<grid, 256, 0, s>>>(static_cast<const uint4*>(d.x), d.d * size / 16, d.d * size / 16, static_cast<uint4*>(p.x), p.x_pitch * size / 16,
                                                       p.rows.index, p.rows.count, d.n, all);
    else if (size == 2)
        gather_rows_kernel<uint16_t><<<grid, 256, 0, s>>>(static_cast<const uint16_t*>(d.x), d.d, d.d, static_cast<uint16_t*>(p.x), p.x_pitch, p.rows.index, p.rows.count,
                                                          d.n, all);
    else
        gather_rows_kernel<uint32_t><<<grid, 256, 0, s>>>(static_cast<const uint32_t*>(d.x), d.d, d.d, static_cast<uint32_t*>(p.x), p.x_pitch, p.rows.index, p.rows.count,
                                                          d.n, all);
    return launch_status();
}

// ---- f32 -------------------------------------------------------------------------------------------------------------------------
// [rows, cols] -> [cols, rows]
int turn(const float* from, int64_t rows, int64_t cols, void* to, cudaStream_t s) {
    const int64_t shape[2] = {cols, rows};
    const int perm[2]      = {1, 0};
    return permute_copy(from, to, 4, 2, shape, perm, s);
}

int run_f32(const mimk_linear_ce_desc& d, const Plan& p, bool forward, bool backward, const DeviceInfo& dev, cudaStream_t s) {
    MIMK_TRY(begin(d, p, forward, dev, s));
    const bool nk      = d.w_layout == MIMK_B_NK;
    const float* x     = static_cast<const float*>(p.x ? p.x : d.x);
    const float* w     = static_cast<const float*>(d.w);
    float *logits      = static_cast<float*>(p.p), *dx = p.dx ? p.dx : static_cast<float*>(d.dx), *dw = static_cast<float*>(d.dw);
    Rows rows          = p.rows;
    for (int64_t first = 0; first < d.n; first += p.piece) {
        const int64_t n = std::min(p.piece, d.n - first);
        const float* xi = x + first * d.d;
        MIMK_TRY(gemm_any(product(n, d.v, d.d, xi, w, d.w_layout, logits), s, p.cut));
        logits_kernel<<<unsigned(n), 512, 0, s>>>(logits, d.v, first, rows, d.dloss, d.reduction, forward ? nullptr : d.lse, forward ? d.lse : nullptr,
                                                  backward);
        MIMK_TRY(launch_status());
        if (!backward) continue;
        MIMK_TRY(gemm_any(product(n, d.d, d.v, logits, w, nk ? MIMK_B_KN : MIMK_B_NK, dx + first * d.d), s, p.cut));
        float* to = first ? static_cast<float*>(p.sum) : dw;
        if (nk) {
            MIMK_TRY(turn(logits, n, d.v, p.turned, s));
            MIMK_TRY(gemm_any(product(d.v, d.d, n, p.turned, xi, MIMK_B_KN, to), s, p.cut));
        } else {
            MIMK_TRY(turn(xi, n, d.d, p.turned, s));
            MIMK_TRY(gemm_any(product(d.d, d.v, n, p.turned, logits, MIMK_B_KN, to), s, p.cut));
        }
        if (first) {
            add_kernel<<<grid_for(d.d * d.v, 1024, 8192), 256, 0, s>>>(dw, to, d.d * d.v);
            MIMK_TRY(launch_status());
        }
    }
    if (forward && d.reduction != MIMK_REDUCTION_NONE) {
        loss_kernel<<<1, 1024, 0, s>>>(rows, d.n, d.reduction, d.loss);
        MIMK_TRY(launch_status());
    }
    if (backward && p.dx) {
        MIMK_TRY(launch_after(place_rows_kernel<float>, grid_for(d.n * ((d.d + 3) / 4), 256, 8192), 256, 0, s, static_cast<const float*>(p.dx), 1, int64_t(0), d.d,
                              static_cast<const int*>(p.rows.place), static_cast<float*>(d.dx), d.n, d.d, false));
    }
    return MIMK_OK;
}

// ---- bf16 ------------------------------------------------------------------------------------------------------------------------
Problem problem(int64_t m, int64_t n, int64_t k, bool a_mn, bool b_mn) {
    Problem p{};
    p.M = int(m), p.N = int(n), p.kb[0] = int((k + BK - 1) / BK), p.a_mn = a_mn, p.b_mn = b_mn, p.splits = 1;
    return p;
}

template <int N, bool GRAD>
int few_rows_of(const mimk_linear_ce_desc& d, const Plan& p, int64_t from, int64_t cols, const DeviceInfo& dev, cudaStream_t s) {
    const int smem = int(N * d.d * 4);
    auto kern      = few_rows_kernel<N, GRAD>;
    if (smem > 48 * 1024) MIMK_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 65536));
    return launch_after(kern, unsigned(dev.sm_count * FEW_CTAS), 256, smem, s, static_cast<const __nv_bfloat16*>(d.x), d.d, static_cast<const __nv_bfloat16*>(d.w) + from * d.d,
                        int(d.d), int(cols), p.rows, int(d.n), int(from), static_cast<__nv_bfloat16*>(p.p), p.piece);
}
// classes [from, from + cols)
template <bool GRAD>
int few_rows(const mimk_linear_ce_desc& d, const Plan& p, int64_t from, int64_t cols, const DeviceInfo& dev, cudaStream_t s) {
    return d.n == 1 ? few_rows_of<1, GRAD>(d, p, from, cols, dev, s) : d.n == 2 ? few_rows_of<2, GRAD>(d, p, from, cols, dev, s) : few_rows_of<FEW, GRAD>(d, p, from, cols, dev, s);
}

int run_bf16(const mimk_linear_ce_desc& d, const Plan& p, bool forward, bool backward, const DeviceInfo& dev, cudaStream_t s) {
    MIMK_TRY(begin(d, p, forward, dev, s));
    MIMK_TRY(stage_in(p.w, s));
    const bool nk    = d.w_layout == MIMK_B_NK;
    const int* count = p.rows.index ? p.rows.count : nullptr;
    const Mat x      = {p.x ? p.x : d.x, d.n, d.d, p.x_pitch};
    const Mat& w     = p.w.use;
    // columns [from, from + cols) of W: rows where it is stored [v, d]
    auto part_of = [&](const Mat& of, int64_t from, int64_t cols) {
        const __nv_bfloat16* at = static_cast<const __nv_bfloat16*>(of.p);
        return nk ? Mat{at + from * of.pitch, cols, of.cols, of.pitch} : Mat{at + from, of.rows, cols, of.pitch};
    };
    Maps maps;
    Args args{};
    args.status = dev.status_dev;
    args.target = p.rows.target, args.lse = p.rows.lse, args.scale = p.rows.scale, args.part = p.rows.part, args.target_logit = p.rows.target_logit;
    float* loss = forward && d.reduction != MIMK_REDUCTION_NONE ? d.loss : nullptr;
    if (forward) {
        args.count      = 1;
        args.p[0]       = problem(d.n, d.v, d.d, false, !nk);
        args.p[0].dyn_m = count;
        if (!p.few) {
            MIMK_TRY(operand_map(&maps.a[0][0], x, false, BM));
            MIMK_TRY(operand_map(&maps.b[0][0], w, !nk, 128));
        }
        if (p.few) {
            MIMK_TRY(few_rows<false>(d, p, 0, d.v, dev, s));
        } else if (p.kept) {
            MIMK_TRY(result_map(&maps.out[0], p.p, false, d.n, d.v, p.piece));
            MIMK_TRY(launch_group<CE_EXP>(maps, args, dev, s));
        } else {
            MIMK_TRY(launch_group<CE_STATS>(maps, args, dev, s));
        }
        MIMK_TRY(launch_after(join_kernel, grid_for(d.n, 1, 4096), 128, 0, s, p.rows, d.n, p.parts, d.dloss, int(d.reduction), loss, d.lse));
    } else {
        recall_kernel<<<grid_for(d.n, 256, 1024), 256, 0, s>>>(p.rows, d.lse, d.dloss, d.reduction);
        MIMK_TRY(launch_status());
    }
    if (!backward) return MIMK_OK;
    if (p.kept) {
        const dim3 grid(unsigned((p.piece + 8191) / 8192), grid_for(d.n, 1, 65535));
        MIMK_TRY(launch_after(probabilities_kernel, grid, 256, 0, s, p.rows, static_cast<uint16_t*>(p.p), p.piece, d.n, p.parts));
    }

    for (int64_t from = 0; from < d.v; from += p.piece) {
        const int64_t cols = std::min(p.piece, d.v - from);
        const Mat wi = part_of(w, from, cols), pi = {p.p, d.n, cols, p.piece};
        if (p.few) {
            MIMK_TRY(few_rows<true>(d, p, from, cols, dev, s));
        } else if (!p.kept) {
            args.count      = 1;
            args.column0    = int(from);
            args.p[0]       = problem(d.n, cols, d.d, false, !nk);
            args.p[0].dyn_m = count;
            MIMK_TRY(operand_map(&maps.a[0][0], x, false, BM));
            MIMK_TRY(operand_map(&maps.b[0][0], wi, !nk, 128));
            MIMK_TRY(result_map(&maps.out[0], p.p, false, d.n, cols, p.piece));
            MIMK_TRY(launch_group<CE_GRAD>(maps, args, dev, s));
        }
        // dx += p W^T: W stored [v, d] has the result's columns contiguous, [d, v] the classes
        args.count      = 2;
        args.p[0]       = problem(d.n, d.d, cols, false, nk);
        args.p[0].dyn_m = count;
        MIMK_TRY(operand_map(&maps.a[0][0], pi, false, BM));
        MIMK_TRY(operand_map(&maps.b[0][0], wi, nk, 128));
        if (p.dx) {
            args.p[0].splits = p.splits, args.p[0].rows_pad = int(p.rows_pad), args.p[0].out_f32 = 1, args.p[0].add = from > 0;
            MIMK_TRY(result_map(&maps.out[0], p.dx, true, p.splits * p.rows_pad, d.d, p.dx_pitch));
        } else {
            MIMK_TRY(result_map(&maps.out[0], d.dx, false, d.n, d.d, d.d));
        }
        // the piece's part of dW: p^T x, or x^T p where W is stored [d, v]
        args.p[1]       = nk ? problem(cols, d.d, d.n, true, true) : problem(d.d, cols, d.n, true, true);
        args.p[1].dyn_k = count;
        MIMK_TRY(operand_map(&maps.a[1][0], nk ? pi : x, true, BM));
        MIMK_TRY(operand_map(&maps.b[1][0], nk ? x : pi, true, 128));
        const Mat out = part_of(p.dw.use, from, cols);
        MIMK_TRY(result_map(&maps.out[1], const_cast<void*>(out.p), false, out.rows, out.cols, out.pitch));
        MIMK_TRY(launch_group<STORE>(maps, args, dev, s));
    }
    MIMK_TRY(stage_out(p.dw, s));
    if (p.dx) {
        const bool words = d.d % 4 == 0 && reinterpret_cast<uintptr_t>(d.dx) % 8 == 0;
        MIMK_TRY(launch_after(place_rows_kernel<__nv_bfloat16>, grid_for(d.n * ((d.d + 3) / 4), 256, 8192), 256, 0, s, static_cast<const float*>(p.dx), p.splits,
                              p.rows_pad * p.dx_pitch, p.dx_pitch, static_cast<const int*>(p.rows.place), static_cast<__nv_bfloat16*>(d.dx), d.n, d.d, words));
    }
    return MIMK_OK;
}

int run(const mimk_linear_ce_desc* d, bool forward, bool backward, void* stream) {
    MIMK_TRY(check(d));
    int st                = MIMK_OK;
    const DeviceInfo* dev = device_info(&st);
    if (!dev) return st;
    cudaStream_t s   = static_cast<cudaStream_t>(stream);
    const bool reduced = d->reduction != MIMK_REDUCTION_NONE;
    if (d->n == 0) {  // no rows: a loss and a gradient of zeros
        if (forward && reduced) {
            if (!d->loss) return MIMK_E_ARG;
            MIMK_CUDA_TRY(cudaMemsetAsync(d->loss, 0, 4, s));
        }
        const size_t cells = size_t(d->d) * size_t(d->v) * dtype_size(d->dtype);
        if (backward && cells) {
            if (!d->dw) return MIMK_E_ARG;
            MIMK_CUDA_TRY(cudaMemsetAsync(d->dw, 0, cells, s));
        }
        return MIMK_OK;
    }
    if (!d->x || !d->w || !d->targets || (forward && !d->loss) || (!forward && !d->lse) || (backward && (!d->dx || !d->dw))) return MIMK_E_ARG;
    Space space(d->workspace);
    const Plan p = plan(*d, forward, backward, space, dev->sm_count);
    if (space.used() > d->workspace_bytes || !d->workspace) return MIMK_E_WORKSPACE;
    if (!aligned16(d->workspace)) return MIMK_E_ALIGN;
    return d->dtype == MIMK_F32 ? run_f32(*d, p, forward, backward, *dev, s) : run_bf16(*d, p, forward, backward, *dev, s);
}

}  // namespace
}  // namespace mimk

using namespace mimk;

extern "C" int mimk_linear_ce_workspace(const mimk_linear_ce_desc* d, int forward, int backward, uint64_t* bytes) {
    MIMK_TRY(check(d));
    if (!bytes || (!forward && !backward)) return MIMK_E_ARG;
    int st                = MIMK_OK;
    const DeviceInfo* dev = device_info(&st);
    if (!dev) return st;
    Space space(nullptr);
    if (d->n > 0) plan(*d, forward != 0, backward != 0, space, dev->sm_count);
    *bytes = space.used();
    return MIMK_OK;
}
extern "C" int mimk_linear_ce_fwd(const mimk_linear_ce_desc* d, void* stream) { return run(d, true, false, stream); }
extern "C" int mimk_linear_ce_bwd(const mimk_linear_ce_desc* d, void* stream) { return run(d, false, true, stream); }
extern "C" int mimk_linear_ce_fwd_bwd(const mimk_linear_ce_desc* d, void* stream) { return run(d, true, true, stream); }
