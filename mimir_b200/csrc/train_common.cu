// Copies between row pitches, and the sum of partial results.
#include "train_common.cuh"

namespace mimk {

namespace {

// Bound by latency or by the bytes; single elements, as either side may start anywhere.
__global__ void copy_rows_kernel(const uint16_t* __restrict__ from, int64_t from_pitch, uint16_t* __restrict__ to, int64_t to_pitch, int64_t rows, int64_t cols) {
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y)
        for (int64_t c = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; c < cols; c += int64_t(gridDim.x) * blockDim.x)
            to[r * to_pitch + c] = from[r * from_pitch + c];
}

// Four columns a thread (the partial results' rows are whole 16 bytes), the parts in order, so that the sum is the same call after call.
__global__ void sum_parts_kernel(const float* part, int splits, int64_t stride, int64_t part_pitch, __nv_bfloat16* out,
                                 int64_t out_pitch, int64_t rows, int64_t cols, bool words) {
    after_previous();
    const int64_t quads = (cols + 3) / 4, all = rows * quads;
    for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < all; i += int64_t(gridDim.x) * blockDim.x) {
        const int64_t r = i / quads, c = (i - r * quads) * 4;
        const float* p = part + r * part_pitch + c;
        float4 v       = *reinterpret_cast<const float4*>(p);
        for (int s = 1; s < splits; ++s) {
            const float4 w = *reinterpret_cast<const float4*>(p + s * stride);
            v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
        }
        __nv_bfloat16* o = out + r * out_pitch + c;
        if (words && c + 4 <= cols) {
            *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
        } else {
            const float e[4] = {v.x, v.y, v.z, v.w};
            for (int j = 0; j < 4 && c + j < cols; ++j) o[j] = __float2bfloat16(e[j]);
        }
    }
}

}  // namespace

int copy_rows(const void* from, int64_t from_pitch, void* to, int64_t to_pitch, int64_t rows, int64_t cols, cudaStream_t s) {
    if (rows <= 0 || cols <= 0) return MIMK_OK;
    const int64_t bx = (cols + 255) / 256;
    const dim3 grid(unsigned(bx < 64 ? bx : 64), unsigned(rows < 16384 ? rows : 16384));
    copy_rows_kernel<<<grid, 256, 0, s>>>(static_cast<const uint16_t*>(from), from_pitch, static_cast<uint16_t*>(to), to_pitch, rows, cols);
    return launch_status();
}

int pick_splits(int64_t m, int64_t n, int64_t kblocks, int sm_count) {
    const int64_t pairs = sm_count / 2, tiles = up(m, 256) / 256 * (up(n, 256) / 256);
    int best         = 1;
    double best_time = 1e300;
    for (int s = 1; s <= 16 && (s == 1 || kblocks / s >= 4); ++s) {
        const double rounds = double((tiles * s + pairs - 1) / pairs);
        double time         = rounds * double((kblocks + s - 1) / s + 6);
        if (s > 1) time += 12 + double(s) * double(m) * double(n) * 8 / 6.5e6 / 0.27;
        if (time < best_time) best = s, best_time = time;
    }
    // (no tile without k-blocks)
    const int64_t per = (kblocks + best - 1) / best;
    return per ? int((kblocks + per - 1) / per) : 1;
}

int sum_parts(const float* part, int splits, int64_t rows_pad, int64_t part_pitch, void* out, int64_t out_pitch, int64_t rows, int64_t cols, cudaStream_t s) {
    const int64_t all = rows * ((cols + 3) / 4), blocks = (all + 255) / 256;
    if (!all) return MIMK_OK;
    const bool words = out_pitch % 4 == 0 && reinterpret_cast<uintptr_t>(out) % 8 == 0;
    return launch_after(sum_parts_kernel, unsigned(blocks < 4096 ? blocks : 4096), 256, 0, s, part, splits, rows_pad * part_pitch, part_pitch, static_cast<__nv_bfloat16*>(out),
                        out_pitch, rows, cols, words);
}

}  // namespace mimk
