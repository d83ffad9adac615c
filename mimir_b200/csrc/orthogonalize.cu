// Orthogonalised updates by Newton-Schulz products. X = x / (|x| + eps); for each step (p, q, r), with k the smaller extent of X and A [k, k]:
//   A = X X^T (X^T X where X is taller than wide),  B = q A + r A^2,  X <- p X + B X (X B)
// Three products a step on the tensor cores. A and B are symmetric: the tiles on and below the diagonal are multiplied, and written twice.
//
// Rounding. Singular values grow by p a step while they are small, and what is rounded away of X grows with them: with all operands in bf16 the result of
// a matrix with falling singular values is off by 5e-2 to 3e-1. Here operands are f16 (11 bits, where bf16 has 8) times powers of two that keep
// their largest possible value below 2^15; p X is added from an X of two f16 (22 bits), so that rounding one operand of B X does not enter X itself;
// and the diagonals of A and B, near which the values of most matrices lie, are kept in f32 and out of the products:
//   with A = O + diag(d):  A^2 = O O + (d_i + d_j) O_ij + diag(d_i^2),  B X = (B - diag(e)) X + diag(e) X
// What the first f16 of X leaves out, L, must not enter the small directions, where it would grow with them: (B - diag(e)) L does, with -e where B has all but nothing (matrices of a few rows and
// hardly any rank came out off by 4e-2, in eight steps by 0.9). Matrices that a CTA takes whole have L multiplied, too. For others diag(e) L is left out as long as singular values can
// still grow by more than 4, so that B L stays in B's own large directions, and is added in the steps from there on, where singular values lie near one another and B near its diagonal.
// Against 64 bits the result, before its own rounding to bf16 (1.66e-3), is off by 2e-4 to 1e-3 for random matrices and such with falling values, and by up to 2.5e-3 for any of some thousand
// spectra and bases tried (nearly parallel rows, two or three levels, a few rows large). With diag(e) L left out of all steps: 1.4e-3 in place of 5e-4 (random, 64 x 256) and
// 2.5e-3; in all but the last three: 4.6e-3; without the second f16 of X 6e-3 to 3e-2 for falling values.
// What bounds it: the tensor cores, where there are many tiles: 4096 x 14336, five steps of k^2 l + k^3 + 2 k^2 l (k <= l) operations: 3.2 ms from idle, 1.24 PFLOP/s, three
// quarters of what a library's product reaches; under the power limit 3.7 ms, 1.06 of 1.40. The tensor cores have work for 0.94 of a tile's time; the rest are
// last rounds of tiles (136 of A and 896 of X over 74 pairs of SMs). Medium sizes: loads from L2, 64 bytes a cycle for each SM (how, below), and the start and end of three dependent launches
// a step, 7 us or more each: 703 x 255 in 125 us, 3 of 1024 x 2816 in 300.
#include <math.h>

#include <cuda_fp16.h>

#include "elements.cuh"
#include "sm100_pair.cuh"
#include "train_common.cuh"

namespace mimk {

namespace {

using namespace sm100;

enum Product {
    GRAM,    // A from X: its values off the diagonal as f16, the diagonal as f32
    SQUARE,  // B from A, the same way
    APPLY,   // the next X from B and X
};
constexpr int BM = 128, BK = 64, OPERAND = BM * BK * 2, STAGE = 2 * OPERAND;
constexpr int FIRST = 3, WARPS = 8, THREADS = (FIRST + WARPS) * 32;  // a warp for each operand's loads and one for the multiplications, then the epilogue's: two for 32 rows
constexpr int SLOT = 4096;  // 32 columns of 32 rows of X, a first and a second f16: two tiles of [32 rows x 64 bytes]
constexpr int GROUP_M = 8;
constexpr float SX = 256.f, LOW = 2048.f;  // factors of X, and of the second f16 of a value against the first

template <int KIND>
struct Shape {
    static constexpr int SLOTS  = KIND == APPLY ? 2 * WARPS : 0;  // two for each warp
    static constexpr int STAGES = KIND == APPLY ? 4 : 6;
    static constexpr int SMEM   = STAGES * STAGE + SLOTS * SLOT + 1024 + 512;
};

struct Maps {
    CUtensorMap left, right, tile, out;  // the last two: tiles of 32 rows and columns of X, and of the result, APPLY
};
struct Args {
    int rows, cols, batch;  // of the result
    int tiles_m, tiles_n, kb;
    int splits, per;  // GRAM: the k-blocks dealt out over that many tiles, `per` each, whose sums are f32 partial results
    int a_mn, b_mn;  // operand stored with its M (N) axis contiguous
    int pitch, diag_pitch;  // of A and B; of the diagonals
    int last, tall;  // APPLY: the result is BF16; e goes with columns
    int z_left, z_right, z_hi, z_lo, z_out_hi, z_out_lo;  // where the batch's matrices begin in the buffers that the maps are of
    const __half* in;  // SQUARE: A
    __half* out;       // GRAM: A, SQUARE: B
    float* part;       // [splits][batch][rows][pitch], tiles on and below the diagonal
    const float* diag_in;  // SQUARE: d, APPLY: e
    float* diag_out;
    // GRAM: A = acc * f[0], times f[4] as f16. SQUARE: O O = acc * f[0], A = in * f[1], q = f[2], r = f[3], times f[4] as f16.
    // APPLY: SX X' = (f[0] + e) SX X + acc * f[1], of X's second f16 only f[3] e; the result times f[2]
    float f[5];
    int* status;
};

struct Bars {
    uint64_t full[6], empty[6], acc_full[2], acc_empty[2], in[2 * WARPS];
    uint32_t tmem_base;
    int abort_flag;
};
static_assert(sizeof(Bars) <= 512, "barrier block too large");

struct Tile {
    int z, m, n, split;
};
template <int KIND, int SIDE>
__device__ __forceinline__ bool tile_at(const Args& g, int index, Tile& t) {
    const int per = KIND == APPLY ? g.tiles_m * g.tiles_n : g.tiles_m * (g.tiles_m + 1) / 2;
    t.split = 0;
    if (KIND == GRAM && g.splits > 1) {
        t.split = index / (per * g.batch), index -= t.split * per * g.batch;
        if (t.split >= g.splits) return false;
    }
    t.z = index / per;
    if (t.z >= g.batch) return false;
    const int i = index - t.z * per;
    if (KIND != APPLY) {
        // row a of the triangle holds tiles a (a + 1) / 2 and on
        int a = int((sqrtf(8.f * float(i) + 1.f) - 1.f) * 0.5f);
        while (a * (a + 1) / 2 > i) --a;
        while ((a + 1) * (a + 2) / 2 <= i) ++a;
        t.m = a * SIDE, t.n = (i - a * (a + 1) / 2) * SIDE;
    } else {
        const int per_group = GROUP_M * g.tiles_n, group = i / per_group, in_group = i - group * per_group;
        const int size = min(g.tiles_m - group * GROUP_M, GROUP_M), column = in_group / size;
        t.m = (group * GROUP_M + in_group - column * size) * SIDE, t.n = column * SIDE;
    }
    return true;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
// 16-byte piece `piece` of this lane's row of a 64-byte-swizzled tile
__device__ __forceinline__ uint32_t piece_at(uint32_t tile, int lane, int piece) { return tile + lane * 64 + ((uint32_t(piece) ^ uint32_t(lane >> 1 & 3)) << 4); }
__device__ __forceinline__ uint4 ld_shared(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void st_shared(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

struct Core {
    uint32_t tile_base, tmem_base;
    Bars* bars;
};
// SMS: 2, a tile of 256 x 256 on a pair of SMs, or 1, one of 128 x 128 on one. A CTA stages 128 rows of the left operand and 128 columns of the right one.
template <int SMS, int STAGES, int SLOTS>
__device__ __forceinline__ Core set_up(uint8_t* smem_raw) {
    const uint32_t raw_addr = smem_u32(smem_raw), tile_base = (raw_addr + 1023u) & ~1023u;
    Core core{tile_base, 0, reinterpret_cast<Bars*>(smem_raw + (tile_base - raw_addr) + STAGES * STAGE + SLOTS * SLOT)};
    Bars* bars = core.bars;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(smem_u32(&bars->full[s]), 1);
            mbar_init(smem_u32(&bars->empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&bars->acc_full[b]), 1);
            mbar_init(smem_u32(&bars->acc_empty[b]), SMS * WARPS * 32);
        }
        for (int w = 0; w < 2 * WARPS; ++w) mbar_init(smem_u32(&bars->in[w]), 1);
        bars->abort_flag = 0;
        fence_barrier_init();
    }
    if (threadIdx.x >> 5 == 1) {
        if constexpr (SMS == 2) {
            tmem_alloc_pair(smem_u32(&bars->tmem_base), 2 * BM * SMS);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(smem_u32(&bars->tmem_base), 2 * BM * SMS);
            tmem_relinquish();
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (SMS == 2) cluster_sync();
    tc_fence_after();
    core.tmem_base = *reinterpret_cast<volatile uint32_t*>(&bars->tmem_base);
    return core;
}
template <int SMS>
__device__ __forceinline__ void tear_down(const Core& core, int* status) {
    tc_fence_before();
    __syncthreads();
    if constexpr (SMS == 2) cluster_sync();  // neither CTA may release shared or tensor memory while the other can still touch it
    if (threadIdx.x >> 5 == 1) {
        __syncwarp();
        tc_fence_after();
        if constexpr (SMS == 2) tmem_dealloc_pair(core.tmem_base, 2 * BM * SMS);
        else tmem_dealloc(core.tmem_base, 2 * BM * SMS);
    }
    if (threadIdx.x == 0 && *const_cast<volatile int*>(&core.bars->abort_flag)) *status = MIMK_E_DEVICE_WAIT;
}

// This CTA's tiles of one product.
template <int KIND, int SMS, int STAGES>
__device__ __forceinline__ void product(const Maps& maps, const Args& g, const Core& core) {
    constexpr int SIDE = BM * SMS, COLUMNS = SIDE;
    const uint32_t tile_base = core.tile_base, tmem_base = core.tmem_base;
    Bars* bars               = core.bars;
    volatile int* abort_flag = &bars->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = SMS == 2 ? cluster_ctarank() : 0;
    const int first = blockIdx.x / SMS, step = gridDim.x / SMS;
    uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0, in_phase = 0;

    Tile t;
    if (warp == 0 || warp == 2) {
        // ---------------- loads: warp 0 the left operand, warp 2 the right one ----------------
        if (lane == 0) {
            const bool left  = warp == 0;
            const int mn     = left ? g.a_mn : g.b_mn;
            const auto* map  = left ? &maps.left : &maps.right;
            const int z0     = left ? g.z_left : g.z_right;
            bool ok = true;
            for (int index = first; ok && tile_at<KIND, SIDE>(g, index, t); index += step) {
                const int at = (left ? t.m : t.n) + int(rank) * BM;
                const int end = KIND == GRAM ? min(g.kb, (t.split + 1) * g.per) : g.kb;
                for (int kb = KIND == GRAM ? t.split * g.per : 0; kb < end; ++kb) {
                    if (!(ok = mbar_wait(smem_u32(&bars->empty[stage]), phase ^ 1u, abort_flag))) break;
                    const uint32_t to = tile_base + stage * STAGE + (left ? 0 : OPERAND), full = smem_u32(&bars->full[stage]);
                    const int k = kb * BK;
                    if (left && rank == 0) mbar_expect_tx(full, SMS * STAGE);
                    if constexpr (SMS == 2) {
                        const uint32_t full_even = map_to_cta(full, 0);
                        if (!mn) {
                            tma_load_3d_pair(to, map, k, at, z0 + t.z, full_even);
                        } else {
                            tma_load_3d_pair(to, map, at, k, z0 + t.z, full_even);
                            tma_load_3d_pair(to + BK * 128, map, at + 64, k, z0 + t.z, full_even);
                        }
                    } else {
                        if (!mn) {
                            tma_load_3d(to, map, k, at, z0 + t.z, full);
                        } else {
                            tma_load_3d(to, map, at, k, z0 + t.z, full);
                            tma_load_3d(to + BK * 128, map, at + 64, k, z0 + t.z, full);
                        }
                    }
                    if (++stage == STAGES) stage = 0, phase ^= 1u;
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- multiplications (of a pair: the even CTA) ----------------
        if (lane == 0 && rank == 0) {
            bool ok = true;
            const uint64_t high  = smem_desc_sw128(0, 0, 1024);
            const uint32_t idesc = idesc_f16_f32(SIDE, SIDE, g.a_mn, g.b_mn);
            // a descriptor's low word is the address >> 4 with the leading offset >> 4 above it, its high word is the same for all
            const uint32_t a_step = g.a_mn ? 2048 >> 4 : 32 >> 4, b_step = g.b_mn ? 2048 >> 4 : 32 >> 4;
            const uint32_t a_low = (g.a_mn ? BK * 128 >> 4 : 1) << 16, b_low = ((g.b_mn ? BK * 128 >> 4 : 1) << 16) + (OPERAND >> 4);
            for (int index = first; ok && tile_at<KIND, SIDE>(g, index, t); index += step) {
                if (!(ok = mbar_wait(smem_u32(&bars->acc_empty[acc]), acc_phase ^ 1u, abort_flag))) break;
                tc_fence_after();
                const int begin = KIND == GRAM ? t.split * g.per : 0, end = KIND == GRAM ? min(g.kb, begin + g.per) : g.kb;
                for (int kb = begin; kb < end; ++kb) {
                    if (!(ok = mbar_wait(smem_u32(&bars->full[stage]), phase, abort_flag))) break;
                    tc_fence_after();
                    const uint32_t at = (tile_base + stage * STAGE) >> 4;
#pragma unroll
                    for (int k = 0; k < BK / 16; ++k) {
                        const uint64_t a = high | (at + a_low + k * a_step), b = high | (at + b_low + k * b_step);
                        if constexpr (SMS == 2) mma_f16_ss_pair(tmem_base + acc * COLUMNS, a, b, idesc, kb > begin || k > 0);
                        else mma_f16_ss(tmem_base + acc * COLUMNS, a, b, idesc, kb > begin || k > 0);
                    }
                    if constexpr (SMS == 2) mma_commit_pair(smem_u32(&bars->empty[stage]));
                    else mma_commit(smem_u32(&bars->empty[stage]));
                    if (++stage == STAGES) stage = 0, phase ^= 1u;
                }
                if (!ok) break;
                if constexpr (SMS == 2) mma_commit_pair(smem_u32(&bars->acc_full[acc]));
                else mma_commit(smem_u32(&bars->acc_full[acc]));
                if (++acc == 2) acc = 0, acc_phase ^= 1u;
            }
        }
    } else {
        // ---------------- epilogue: 32 rows and half of the columns for each warp, a row per lane ----------------
        constexpr int HALF = SIDE / 2;
        const int quarter = warp & 3, half = (warp - FIRST) >> 2, side = half * HALF;
        const uint32_t slot = tile_base + STAGES * STAGE + (warp - FIRST) * 2 * SLOT, in_bar = smem_u32(&bars->in[(warp - FIRST) * 2]);
        bool ok   = true;
        bool have = tile_at<KIND, SIDE>(g, first, t);
        // APPLY: 32 columns of X, in two sets of slots in turn
        auto request = [&](int c) {
            const int row = t.m + int(rank) * BM + quarter * 32;
            if (KIND == APPLY && lane == 0 && row < g.rows && c < side + HALF && t.n + c < g.cols) {
                const uint32_t set = c >> 5 & 1, to = slot + set * SLOT, bar = in_bar + set * 8;
                mbar_expect_tx(bar, SLOT);
                tma_load_3d(to, &maps.tile, t.n + c, row, g.z_hi + t.z, bar);
                tma_load_3d(to + SLOT / 2, &maps.tile, t.n + c, row, g.z_lo + t.z, bar);
            }
        };
        if (have) request(side), request(side + 32);
        for (int index = first; have && ok;) {
            const int row0 = t.m + int(rank) * BM + quarter * 32, row = row0 + lane, end = min(side + HALF, g.cols - t.n);
            const bool there = row < g.rows;
            // SQUARE: A's values, and the diagonal's of their columns, 32 columns asked for ahead
            const int64_t matrix = int64_t(t.z) * g.rows;  // (rows of the matrices before this one)
            const float* diag    = g.diag_in + int64_t(t.z) * g.diag_pitch;
            uint4 a[4];
            float4 dj[8];
            auto ask = [&](int c) {
                if constexpr (KIND == SQUARE) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        a[i] = there && t.n + c + 8 * i < g.cols ? __ldcg(reinterpret_cast<const uint4*>(g.in + (matrix + row) * g.pitch + t.n + c + 8 * i)) : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 8; ++i) dj[i] = t.n + c + 4 * i < g.cols ? __ldcg(reinterpret_cast<const float4*>(diag + t.n + c + 4 * i)) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
            };
            if (row0 < g.rows && side < end) ask(side);
            const float d = KIND == SQUARE && there ? __ldcg(diag + row) : 0.f;
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars->acc_full[acc]), acc_phase, abort_flag)))) break;
            tc_fence_after();
            const uint32_t from = tmem_base + acc * COLUMNS + (uint32_t(quarter * 32) << 16);
            const uint32_t acc_empty = SMS == 2 ? map_to_cta(smem_u32(&bars->acc_empty[acc]), 0) : smem_u32(&bars->acc_empty[acc]);
            if (++acc == 2) acc = 0, acc_phase ^= 1u;
            auto release = [&] {
                tc_fence_before();
                if constexpr (SMS == 2) mbar_arrive_cluster(acc_empty);
                else mbar_arrive(acc_empty);
            };
            if (row0 >= g.rows || side >= end) {
                release();
            } else if constexpr (KIND != APPLY) {
                __half* out = g.out + matrix * g.pitch;
                float* part = g.part + (int64_t(t.split) * g.batch * g.rows + matrix + row) * g.pitch + t.n;
#pragma unroll 1
                for (int c = side; c < end; c += 32) {
                    uint32_t raw[32];
                    tmem_ld_32x32(from + c, raw);
                    tmem_ld_wait();
                    if (c + 32 >= end) release();
                    if (KIND == GRAM && g.splits > 1) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            if (there && t.n + c + i < g.cols) *reinterpret_cast<uint4*>(part + c + i) = make_uint4(raw[i], raw[i + 1], raw[i + 2], raw[i + 3]);
                        continue;
                    }
                    float v[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(raw[i]) * g.f[0];
                    if constexpr (KIND == SQUARE) {
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const float2 o = unpack_f16((&a[i >> 3].x)[i >> 1 & 3]);
                            const float d0 = (&dj[i >> 2].x)[i & 3], d1 = (&dj[i >> 2].x)[(i & 3) + 1];
                            v[i]     = fmaf(fmaf(g.f[3], d + d0, g.f[2]), o.x * g.f[1], g.f[3] * v[i]);
                            v[i + 1] = fmaf(fmaf(g.f[3], d + d1, g.f[2]), o.y * g.f[1], g.f[3] * v[i + 1]);
                        }
                    }
                    if (row0 == t.n + c) {  // the diagonal: lane i has it in column i
                        float on = 0.f;
#pragma unroll
                        for (int i = 0; i < 32; ++i) on = i == lane ? __uint_as_float(raw[i]) * g.f[0] : on, v[i] = i == lane ? 0.f : v[i];
                        if (KIND == SQUARE) on = g.f[2] * d + g.f[3] * fmaf(d, d, on);
                        if (there) g.diag_out[int64_t(t.z) * g.diag_pitch + row] = on;
                    }
                    if (c + 32 < end) ask(c + 32);
                    uint32_t two[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) two[i] = pack_f16(v[2 * i] * g.f[4], v[2 * i + 1] * g.f[4]);
                    if (there) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (t.n + c + 8 * i < g.cols)
                                *reinterpret_cast<uint4*>(out + int64_t(row) * g.pitch + t.n + c + 8 * i) = make_uint4(two[4 * i], two[4 * i + 1], two[4 * i + 2], two[4 * i + 3]);
                    }
                    if (t.m != t.n) {
                        // the other triangle: an even lane stores its row's and the next one's value of an even column, an odd lane those of the odd column
                        const bool odd = lane & 1;
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const uint32_t other = __shfl_xor_sync(0xffffffffu, two[i], 1);
                            const uint32_t both  = odd ? __byte_perm(other, two[i], 0x7632) : __byte_perm(two[i], other, 0x5410);
                            const int column = t.n + c + 2 * i + odd, pair = row & ~1;
                            if (column < g.cols && pair < g.rows) {
                                __half* to = out + int64_t(column) * g.pitch + pair;
                                *reinterpret_cast<uint32_t*>(to) = both;  // (a last odd row's neighbour lies in the rows' padding)
                            }
                        }
                    }
                }
            } else {
                const float e = !g.tall && there ? __ldcg(diag + row) : 0.f;
#pragma unroll 1
                for (int c = side; c < end; c += 32) {
                    const uint32_t set = c >> 5 & 1, at = slot + set * SLOT;
                    if (!(ok = __all_sync(0xffffffffu, mbar_wait(in_bar + set * 8, in_phase >> set & 1u, abort_flag)))) break;
                    in_phase ^= 1u << set;
                    uint32_t raw[32];
                    tmem_ld_32x32(from + c, raw);
                    float4 ej[8];
                    if (g.tall) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) ej[i] = t.n + c + 4 * i < g.cols ? __ldcg(reinterpret_cast<const float4*>(diag + t.n + c + 4 * i)) : make_float4(0.f, 0.f, 0.f, 0.f);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) ej[i] = make_float4(e, e, e, e);
                    }
                    uint4 hi[4], lo[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) hi[i] = ld_shared(piece_at(at, lane, i)), lo[i] = ld_shared(piece_at(at + SLOT / 2, lane, i));
                    tmem_ld_wait();
                    if (c + 32 >= end) release();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t h[4] = {hi[i].x, hi[i].y, hi[i].z, hi[i].w}, l[4] = {lo[i].x, lo[i].y, lo[i].z, lo[i].w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int k    = 8 * i + 2 * j;
                            const float2 a = unpack_f16(h[j]), b = unpack_f16(l[j]);
                            const float e0 = (&ej[k >> 2].x)[k & 3], e1 = (&ej[k >> 2].x)[(k & 3) + 1];
                            const float x = fmaf(g.f[0] + e0, a.x, fmaf(fmaf(g.f[3], e0, g.f[0]) * (1.f / LOW), b.x, __uint_as_float(raw[k]) * g.f[1]));
                            const float y = fmaf(g.f[0] + e1, a.y, fmaf(fmaf(g.f[3], e1, g.f[0]) * (1.f / LOW), b.y, __uint_as_float(raw[k + 1]) * g.f[1]));
                            if (g.last) {
                                h[j] = pack_bf16x2(x * g.f[2], y * g.f[2]);
                            } else {
                                h[j] = pack_f16(x, y);
                                const float2 r = unpack_f16(h[j]);
                                l[j] = pack_f16((x - r.x) * LOW, (y - r.y) * LOW);
                            }
                        }
                        st_shared(piece_at(at, lane, i), h[0], h[1], h[2], h[3]);
                        if (!g.last) st_shared(piece_at(at + SLOT / 2, lane, i), l[0], l[1], l[2], l[3]);
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_3d(&maps.out, at, t.n + c, row0, g.z_out_hi + t.z);
                        if (!g.last) tma_store_3d(&maps.out, at + SLOT / 2, t.n + c, row0, g.z_out_lo + t.z);
                        bulk_commit();
                        if (c > side) bulk_wait_read_1();
                    }
                    if (c > side) request(c + 32);  // (into the set of the columns before these, whose store has been read)
                }
                if (lane == 0) bulk_wait_read_0();
                if (!ok) break;
            }
            index += step;
            have = tile_at<KIND, SIDE>(g, index, t);
            if (have) request(side), request(side + 32);
        }
        if (KIND == APPLY && lane == 0) bulk_wait_all();
    }
}
template <int KIND, int SMS>
__device__ __forceinline__ void one_product(const Maps& maps, const Args& g) {
    extern __shared__ uint8_t smem_raw[];
    if (threadIdx.x == 32) {
        tma_prefetch_desc(&maps.left), tma_prefetch_desc(&maps.right);
        if (KIND == APPLY) tma_prefetch_desc(&maps.tile), tma_prefetch_desc(&maps.out);
    }
    const Core core = set_up<SMS, Shape<KIND>::STAGES, Shape<KIND>::SLOTS>(smem_raw);
    after_previous();
    product<KIND, SMS, Shape<KIND>::STAGES>(maps, g, core);
    tear_down<SMS>(core, g.status);
}
template <int KIND>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1) pair_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args g) {
    one_product<KIND, 2>(maps, g);
}
template <int KIND>
__global__ void __launch_bounds__(THREADS, 1) single_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args g) {
    one_product<KIND, 1>(maps, g);
}

// A from partial results: 8 rows and 32 columns of it for each warp, a column per lane; on and below the diagonal, and the other triangle's from there.
__global__ void __launch_bounds__(256) sum_kernel(const __grid_constant__ Args g, int splits) {
    after_previous();
    const int lane = threadIdx.x & 31, across = (g.cols + 31) / 32, down = (g.rows + 7) / 8;
    const int64_t stride = int64_t(g.batch) * g.rows * g.pitch, units = int64_t(across) * down;
    for (int64_t u = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5); u < units * g.batch; u += int64_t(gridDim.x) * 8) {
        const int z = int(u / units), i = int(u - z * units), row0 = i / across * 8, column0 = i % across * 32, column = column0 + lane;
        if (row0 + 7 < column0) continue;
        const int64_t matrix = int64_t(z) * g.rows;
        const float* p = g.part + (matrix + row0) * g.pitch + column;
        float v[8] = {};
#pragma unroll 2
        for (int s = 0; s < splits; ++s)
#pragma unroll
            for (int r = 0; r < 8; ++r) v[r] += column < g.cols && row0 + r < g.rows ? __ldcg(p + s * stride + r * g.pitch) : 0.f;
        __half h[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            v[r] *= g.f[0];
            if (row0 + r == column && column < g.cols) g.diag_out[int64_t(z) * g.diag_pitch + column] = v[r], v[r] = 0.f;
            h[r] = __float2half_rn(v[r] * g.f[4]);
            if (column <= row0 + r && column < g.cols && row0 + r < g.rows) g.out[(matrix + row0 + r) * g.pitch + column] = h[r];
        }
        __half* other = g.out + (matrix + column) * g.pitch + row0;
        if (column0 + 31 < row0 && row0 + 8 <= g.rows) {
            *reinterpret_cast<uint4*>(other) = *reinterpret_cast<const uint4*>(h);
        } else {
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (column < row0 + r && column < g.cols && row0 + r < g.rows) other[r] = h[r];
        }
    }
}

// ---- x to X ----------------------------------------------------------------------------------------------------------------------
constexpr int TABLE = 1024;       // matrices of one launch
constexpr int PREPARE = 256;
// Values that one block squares: eight for each thread, more where that would be more than some 1200 blocks.
__host__ __device__ __forceinline__ int64_t chunk_of(int64_t count) { return (count / 1184 + 8 * PREPARE) / (8 * PREPARE) * (8 * PREPARE); }

struct Matrices {
    const void* x[TABLE];
};

__device__ __forceinline__ double block_total(double v) {
    __shared__ double part[PREPARE / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < PREPARE / 32; ++w) v += part[w];
    return v;
}
// Eight squares in f32, or in f64 where they overflow or all but vanish
template <int VEC>
__device__ __forceinline__ double squares(const float (&v)[VEC]) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < VEC; ++j) s = fmaf(v[j], v[j], s);
    if (s > 1e-25f && s < INFINITY) return double(s);
    double d = 0;
#pragma unroll
    for (int j = 0; j < VEC; ++j) d += double(v[j]) * double(v[j]);
    return d;
}
// SX / (norm + eps), in two factors, as one may be beyond f32; NaN of a norm that is not finite, zero (for zeros to stay so) where norm and eps are zero
struct Inverse {
    float first, second;
    __device__ __forceinline__ Inverse(double norm, float eps) {
        const double by = !isfinite(norm) ? double(NAN) : norm + double(eps) > 0 ? 1.0 / (norm + double(eps)) : 0.0;
        int power         = 0;
        const double lead = isfinite(by) ? frexp(by, &power) : by;
        first = ldexpf(1.f, power / 2), second = float(ldexp(lead, power - power / 2)) * SX;
    }
    __device__ __forceinline__ float times(float v) const { return v * first * second; }
};
template <class T, int VEC>
__global__ void __launch_bounds__(PREPARE) squares_kernel(const __grid_constant__ Matrices all, int64_t count, double* sums) {
    after_previous();
    const T* x           = static_cast<const T*>(all.x[blockIdx.y]);
    const int64_t chunk  = chunk_of(count), begin = blockIdx.x * chunk, end = min(count, begin + chunk);
    double sum           = 0;
#pragma unroll 8
    for (int64_t i = begin + threadIdx.x * VEC; i < end; i += PREPARE * VEC) {
        Run<T, VEC> run;
        float v[VEC];
        run.load(x + i), run.get(v);
        sum += squares(v);
    }
    sum = block_total(sum);
    if (threadIdx.x == 0) sums[blockIdx.y * gridDim.x + blockIdx.x] = sum;
}
// X times SX as two f16: rows of `pitch`. Every block adds the chunks' sums up itself, in the same order.
template <class T, int VEC>
__global__ void __launch_bounds__(PREPARE) prepare_kernel(const __grid_constant__ Matrices all, int rows, int cols, int pitch, const double* sums, float eps, __half* hi, __half* lo) {
    after_previous();
    const int64_t count = int64_t(rows) * cols;
    const int chunks    = int((count + chunk_of(count) - 1) / chunk_of(count));
    double total        = 0;
    for (int i = threadIdx.x; i < chunks; i += PREPARE) total += sums[blockIdx.y * chunks + i];
    const Inverse by(sqrt(block_total(total)), eps);
    const T* x          = static_cast<const T*>(all.x[blockIdx.y]);
    const int64_t base  = int64_t(blockIdx.y) * rows * pitch;
    const int units     = (cols + VEC - 1) / VEC;  // of a row
    int log             = 0;                       // a row to 2^log threads
    while (log < 8 && 1 << log < units) ++log;
    const int together = PREPARE >> log;
    for (int row = blockIdx.x * together + (threadIdx.x >> log); row < rows; row += gridDim.x * together)
#pragma unroll 2
        for (int u = threadIdx.x & ((1 << log) - 1); u < units; u += 1 << log) {
            Run<T, VEC> run;
            float v[VEC];
            run.load(x + int64_t(row) * cols + u * VEC), run.get(v);
            __half h[VEC], l[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                v[j] = by.times(v[j]);
                h[j] = __float2half_rn(v[j]), l[j] = __float2half_rn((v[j] - __half2float(h[j])) * LOW);
            }
            const int64_t at = base + int64_t(row) * pitch + u * VEC;
            if constexpr (VEC == 8) {
                *reinterpret_cast<uint4*>(hi + at) = *reinterpret_cast<const uint4*>(h);
                *reinterpret_cast<uint4*>(lo + at) = *reinterpret_cast<const uint4*>(l);
            } else {
                hi[at] = h[0], lo[at] = l[0];
            }
        }
}

// ---- small matrices --------------------------------------------------------------------------------------------------------------
// All steps of a matrix with up to 128 rows and 256 columns (or turned: 256 and 128) in one CTA: X as f32 in tensor memory and as two f16 in shared memory, 64 columns to a
// 128-byte row, of which the first serves as the operand of X X^T and both as the right one of B X; A, then B, as f16 in another such matrix. Eight warps: 32 rows, one to a lane, and half of
// the columns each. A step of [128, 128] takes 5 us: its three products 900 cycles each (issued by one thread), the rest what is between them. 64 matrices: 27 us a call
// among others, 34 with cold caches (30 without X's second f16; 141 by launches of their own for each product, from which matrices that do not fit here are taken).
constexpr int SMALL_K = 128, SMALL_L = 256, SMALL_THREADS = 256, CHUNK64 = 128 * 128;  // bytes of 128 rows of 64 columns
constexpr int MOST_STEPS = 64;
struct Factors {
    float p, q, r, a, b;  // a step's coefficients, and the factors of A and B
    float low;            // 1: diag(B) times X's second f16 is added, 0: not (matrices that a CTA does not take whole)
};
struct SmallArgs {
    int k, l, chunks, steps;  // rows and columns of X (turned where x is taller than wide), its chunks of 64 columns
    int vec;                  // rows of x and of the result are whole 16 bytes
    float eps, scale;
    __nv_bfloat16* out;
    int* status;
    Factors f[MOST_STEPS];
};
struct SmallShared {
    uint64_t done;
    uint32_t tmem_base;
    int abort_flag;
    alignas(16) float d[SMALL_K];
    float e[SMALL_K];
    double part[SMALL_THREADS / 32];
};
// 16-byte piece of row `row` of a 128-byte-swizzled matrix of 64-column chunks
__device__ __forceinline__ uint32_t at64(uint32_t base, int row, int column) {
    return base + (column >> 6) * CHUNK64 + row * 128 + ((uint32_t(column >> 3 & 7) ^ uint32_t(row & 7)) << 4);
}
__device__ __forceinline__ void put_tmem(uint32_t to, const float (&v)[32]) {
#pragma unroll
    for (int h = 0; h < 32; h += 16) {
        uint32_t r[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(v[h + i]);
        tmem_st_32x32_x16(to + h, r);
    }
}
// 32 values of X's row as f16, and what that leaves out of them as another (as it is: X is SX times values up to 1, of 1 / 181 and more on the average, whose 12th to 23rd bits lie above 2^-24)
__device__ __forceinline__ void put_x(uint32_t first, uint32_t second, int row, int column, const float (&v)[32]) {
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
        uint32_t h[4], l[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            h[j] = pack_f16(v[i + 2 * j], v[i + 2 * j + 1]);
            const float2 r = unpack_f16(h[j]);
            l[j] = pack_f16(v[i + 2 * j] - r.x, v[i + 2 * j + 1] - r.y);
        }
        st_shared(at64(first, row, column + i), h[0], h[1], h[2], h[3]);
        st_shared(at64(second, row, column + i), l[0], l[1], l[2], l[3]);
    }
}
// 32 values of a row as f16
__device__ __forceinline__ void put_row(uint32_t base, int row, int column, const float (&v)[32], float by) {
#pragma unroll
    for (int i = 0; i < 32; i += 8)
        st_shared(at64(base, row, column + i), pack_f16(v[i] * by, v[i + 1] * by), pack_f16(v[i + 2] * by, v[i + 3] * by), pack_f16(v[i + 4] * by, v[i + 5] * by), pack_f16(v[i + 6] * by, v[i + 7] * by));
}

template <class T, bool TALL>
__global__ void __launch_bounds__(SMALL_THREADS) small_kernel(const __grid_constant__ Matrices all, const __grid_constant__ SmallArgs g) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ SmallShared sh;
    const uint32_t raw = smem_u32(smem_raw), x16 = (raw + 1023u) & ~1023u, a16 = x16 + g.chunks * CHUNK64, low16 = a16 + 2 * CHUNK64;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = (warp & 3) * 32 + lane, half = warp >> 2;
    const int width = g.chunks * 64, columns = g.chunks > 2 ? 512 : 256;  // of tensor memory: X, and the products behind it
    if (threadIdx.x == 0) mbar_init(smem_u32(&sh.done), 1), sh.abort_flag = 0, fence_barrier_init();
    if (warp == 0) {
        tmem_alloc(smem_u32(&sh.tmem_base), columns);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&sh.tmem_base) + (uint32_t((warp & 3) * 32) << 16), acc = tmem + columns / 2;
    const uint32_t mma_acc = *reinterpret_cast<volatile uint32_t*>(&sh.tmem_base) + columns / 2;
    after_previous();

    // x, its columns from `half` of them on
    const T* x       = static_cast<const T*>(all.x[blockIdx.x]);
    const bool there = row < g.k;
    double total     = 0;
#pragma unroll 1
    for (int c = half * width / 2; c < (half + 1) * width / 2; c += 32) {
        float v[32];
        if (!TALL && g.vec) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
                Run<T, 8> run;
                run.clear();
                if (there && c + i < g.l) run.load(x + int64_t(row) * g.l + c + i);
                run.get(*reinterpret_cast<float(*)[8]>(v + i));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                Run<T, 1> run;
                run.clear();
                if (there && c + i < g.l) run.load(TALL ? x + int64_t(c + i) * g.k + row : x + int64_t(row) * g.l + c + i);
                run.get(*reinterpret_cast<float(*)[1]>(v + i));
            }
        }
#pragma unroll
        for (int i = 0; i < 32; i += 8) total += squares(*reinterpret_cast<const float(*)[8]>(v + i));
        put_tmem(tmem + c, v);
    }
    tmem_st_wait();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane == 0) sh.part[warp] = total;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < SMALL_THREADS / 32; ++w) total += sh.part[w];
    const Inverse by(sqrt(total), g.eps);
#pragma unroll 1
    for (int c = half * width / 2; c < (half + 1) * width / 2; c += 32) {
        uint32_t r[32];
        float v[32];
        tmem_ld_32x32(tmem + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = by.times(__uint_as_float(r[i]));
        put_tmem(tmem + c, v);
        put_x(x16, low16, row, c, v);
    }
    tmem_st_wait();

    uint32_t phase = 0;
    bool ok        = true;
    // What is in shared memory is multiplied by one thread, `issue`, and all wait for the result.
    auto multiply = [&](auto&& issue) {
        fence_proxy_async_smem();
        tc_fence_before();
        __syncthreads();
        if (threadIdx.x == 0) {
            tc_fence_after();
            issue();
            mma_commit(smem_u32(&sh.done));
        }
        ok = mbar_wait(smem_u32(&sh.done), phase, &sh.abort_flag);
        phase ^= 1u;
        __syncwarp();
        tc_fence_after();
    };
    const uint64_t high  = smem_desc_sw128(0, 0, 1024);
    const int kblocks    = (g.k + 63) / 64;
    const uint32_t square = idesc_f16_f32(128, 128, 0, 0), wide = idesc_f16_f32(128, width, 0, 1);
    for (int step = 0; step < g.steps; ++step) {
        const Factors f = g.f[step];
        const bool last = step + 1 == g.steps;
        uint32_t both[2][32];
        // A
        multiply([&] {
            for (int c = 0; c < g.chunks; ++c)
                for (int i = 0; i < 4; ++i) {
                    const uint64_t d = high | (((x16 + c * CHUNK64 + i * 32) >> 4) | 1u << 16);
                    mma_f16_ss(mma_acc, d, d, square, c > 0 || i > 0);
                }
        });
        tmem_ld_32x32(acc + half * 64, both[0]);
        tmem_ld_32x32(acc + half * 64 + 32, both[1]);
        tmem_ld_wait();
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            const int c = half * 64 + part * 32;
            uint32_t(&r)[32] = both[part];
            float v[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]) * (1.f / (SX * SX));
            if (c == (warp & 3) * 32) {  // the diagonal: lane i has it in column i
                float on = 0.f;
#pragma unroll
                for (int i = 0; i < 32; ++i) on = i == lane ? v[i] : on, v[i] = i == lane ? 0.f : v[i];
                sh.d[row] = on;
            }
            put_row(a16, row, c, v, f.a);
        }
        // B
        multiply([&] {
            for (int c = 0; c < kblocks; ++c)
                for (int i = 0; i < 4; ++i) {
                    const uint64_t d = high | (((a16 + c * CHUNK64 + i * 32) >> 4) | 1u << 16);
                    mma_f16_ss(mma_acc, d, d, square, c > 0 || i > 0);
                }
        });
        const float di = sh.d[row], less = 1.f / f.a;
        tmem_ld_32x32(acc + half * 64, both[0]);
        tmem_ld_32x32(acc + half * 64 + 32, both[1]);
        tmem_ld_wait();
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            const int c = half * 64 + part * 32;
            uint32_t(&r)[32] = both[part];
            float v[32];
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
                const uint4 w = ld_shared(at64(a16, row, c + i));
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const float2 o = unpack_f16((&w.x)[j >> 1]);
                    const float2 dj = *reinterpret_cast<const float2*>(&sh.d[c + i + j]);
                    v[i + j]     = fmaf(fmaf(f.r, di + dj.x, f.q), o.x * less, f.r * (__uint_as_float(r[i + j]) * less * less));
                    v[i + j + 1] = fmaf(fmaf(f.r, di + dj.y, f.q), o.y * less, f.r * (__uint_as_float(r[i + j + 1]) * less * less));
                }
            }
            if (c == (warp & 3) * 32) {
                float on = 0.f;
#pragma unroll
                for (int i = 0; i < 32; ++i) on = i == lane ? __uint_as_float(r[i]) : on, v[i] = i == lane ? 0.f : v[i];
                sh.e[row] = f.q * di + f.r * fmaf(di, di, on * less * less);
            }
            put_row(a16, row, c, v, f.b);
        }
        // X
        multiply([&] {
            for (const uint32_t x : {x16, low16})
                for (int c = 0; c < kblocks; ++c)
                    for (int i = 0; i < 4; ++i)
                        mma_f16_ss(mma_acc, high | (((a16 + c * CHUNK64 + i * 32) >> 4) | 1u << 16), high | (((x + (c * 64 + i * 16) * 128) >> 4) | uint32_t(CHUNK64 >> 4) << 16), wide,
                                   x == low16 || c > 0 || i > 0);
        });
        const float plus = f.p + sh.e[row], back = 1.f / f.b;
        __nv_bfloat16* out = g.out + int64_t(blockIdx.x) * g.k * g.l;
#pragma unroll 1
        for (int c = half * width / 2; c < (half + 1) * width / 2; c += 32) {
            uint32_t r[32], was[32];
            float v[32];
            tmem_ld_32x32(acc + c, r);
            tmem_ld_32x32(tmem + c, was);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = fmaf(plus, __uint_as_float(was[i]), __uint_as_float(r[i]) * back);
            if (!last) {
                put_tmem(tmem + c, v);
                put_x(x16, low16, row, c, v);
                continue;
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] *= g.scale * (1.f / SX);
            if (!there) continue;
            if (!TALL && g.vec) {
#pragma unroll
                for (int i = 0; i < 32; i += 8)
                    if (c + i < g.l) put(out + int64_t(row) * g.l + c + i, *reinterpret_cast<const float(*)[8]>(v + i));
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (c + i < g.l) out[TALL ? int64_t(c + i) * g.k + row : int64_t(row) * g.l + c + i] = __float2bfloat16(v[i]);
            }
        }
        tmem_st_wait();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(*reinterpret_cast<volatile uint32_t*>(&sh.tmem_base), columns);
    }
    if (threadIdx.x == 0 && !ok) *g.status = MIMK_E_DEVICE_WAIT;
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
using Desc = mimk_orthogonalize_desc;
constexpr int64_t LIM = int64_t(1) << 24, SLICE = int64_t(1) << 30;
// The largest |p v + q v^3 + r v^5| for v from 0 to `most`: there, or where the derivative p + 3 q u + 5 r u^2 is zero, u = v^2. (On the host in every call: 4097 values of v took 12 us a step, a
// call for 64 of 128 x 128 33 us with nothing else to wait for.)
double largest(double p, double q, double r, double most) {
    double found    = 0;
    const auto take = [&](double u) {
        if (!(u > 0 && u <= most * most)) return;
        const double v = fabs(sqrt(u) * (p + u * (q + r * u)));
        if (v > found) found = v;
    };
    take(most * most);
    const double under = 9 * q * q - 20 * p * r;
    if (under >= 0) {
        // (both roots without a difference of like numbers: t / 5r and p / t)
        const double t = -0.5 * (3 * q + (q < 0 ? -sqrt(under) : sqrt(under)));
        if (r != 0) take(t / (5 * r));
        if (t != 0) take(p / t);
    }
    return found;
}
// Every step's factors: powers of two that keep what A and B can hold below 2^15, from the largest singular value that there can be (with a hundredth for what the products round).
int factors_of(const Desc& d, Factors (&f)[MOST_STEPS]) {
    double most = 1;
    for (int s = 0; s < d.steps; ++s) {
        const double p = d.coefficients[3 * s], q = d.coefficients[3 * s + 1], r = d.coefficients[3 * s + 2];
        if (!(fabs(p) <= 1e4 && fabs(q) <= 1e4 && fabs(r) <= 1e4)) return MIMK_E_UNSUPPORTED;
        const double a = most * most, b = fabs(q) * a + fabs(r) * a * a;
        const auto power = [](double v) { return float(exp2(floor(log2(32768.0 / (v > 1.0 / 1024 ? v : 1.0 / 1024))))); };
        f[s] = {float(p), float(q), float(r), power(a), power(b), 0.f};
        most = 1.01 * largest(p, q, r, most);
        if (!(most <= 4)) return MIMK_E_UNSUPPORTED;
        if (most < 1e-3) most = 1e-3;
    }
    // by how much small singular values grow in the steps that follow
    double growth = 1;
    for (int s = d.steps - 1; s >= 0; --s) f[s].low = growth <= 4 ? 1.f : 0.f, growth *= fabs(double(d.coefficients[3 * s]));
    return MIMK_OK;
}

int check(const Desc* d) {
    if (!d || d->batch < 0 || d->m < 0 || d->n < 0 || d->steps < 1 || !d->coefficients || (d->batch && !d->x)) return MIMK_E_ARG;
    if (d->dtype != MIMK_F32 && d->dtype != MIMK_BF16) return MIMK_E_DTYPE;
    if (!(d->eps >= 0)) return MIMK_E_ARG;
    if (d->steps > MOST_STEPS || d->m >= LIM || d->n >= LIM || d->batch >= LIM || d->m * d->n >= (int64_t(1) << 40)) return MIMK_E_UNSUPPORTED;
    return MIMK_OK;
}
bool nothing(const Desc& d) { return !d.batch || !d.m || !d.n; }

struct Plan {
    int64_t k, pitch_x, pitch_a, pitch_d, slice, chunks;
    __half *x[2][2], *a, *b;
    float *d, *e;
    double* sums;
    int splits;          // partial results of A that there is room for
    float* part;
    __nv_bfloat16* out;  // rows of pitch_x, where the result's are no whole 16 bytes
};
Plan plan(const Desc& d, Space& space) {
    Plan p{};
    p.k = d.m < d.n ? d.m : d.n, p.pitch_x = up(d.n, 8), p.pitch_a = up(p.k, 8), p.pitch_d = up(p.k, 4);
    p.chunks = (d.m * d.n + chunk_of(d.m * d.n) - 1) / chunk_of(d.m * d.n);
    // Partial results where A has few tiles and they are long: no more bytes than X has.
    const int64_t l = d.m < d.n ? d.n : d.m, part = 4 * p.k * p.pitch_a;
    p.splits = 1;
    while (p.splits < 64 && p.splits * 2 * part <= 8 * d.m * p.pitch_x && p.splits * 2 * BK * 4 <= l) p.splits *= 2;
    const int64_t each = 8 * d.m * p.pitch_x + 4 * p.k * p.pitch_a + (p.splits > 1 ? p.splits * part : 0);
    p.slice = SLICE / each;
    if (p.slice > d.batch) p.slice = d.batch;
    if (p.slice > TABLE) p.slice = TABLE;
    if (p.slice < 1) p.slice = 1;
    // one after another: the four of X, A and B
    __half* x = static_cast<__half*>(space.take(size_t(4 * p.slice * d.m * p.pitch_x) * 2));
    for (int i = 0; i < 4; ++i) p.x[i >> 1][i & 1] = x ? x + i * p.slice * d.m * p.pitch_x : nullptr;
    p.a = static_cast<__half*>(space.take(size_t(2 * p.slice * p.k * p.pitch_a) * 2)), p.b = p.a ? p.a + p.slice * p.k * p.pitch_a : nullptr;
    p.d = static_cast<float*>(space.take(size_t(p.slice * p.pitch_d) * 4)), p.e = static_cast<float*>(space.take(size_t(p.slice * p.pitch_d) * 4));
    if (p.splits > 1) p.part = static_cast<float*>(space.take(size_t(p.slice) * size_t(p.splits) * size_t(part)));
    p.sums = static_cast<double*>(space.take(size_t(p.slice * p.chunks) * 8));
    // the same for every address of the result (a size is asked for before there is one)
    p.out = static_cast<__nv_bfloat16*>(space.take(size_t(p.slice * d.m * p.pitch_x) * 2));
    return p;
}

int map_of(CUtensorMap* map, const void* p, int64_t rows, int64_t cols, int64_t pitch, int64_t batch, int box) {
    return make_tmap_bf16_3d(map, p, uint64_t(cols), uint64_t(rows), uint64_t(batch), uint64_t(pitch) * 2, uint64_t(rows * pitch) * 2, 64, uint32_t(box));
}

int tile_map(CUtensorMap* map, const void* p, int64_t rows, int64_t cols, int64_t pitch, int64_t batch) {
    const cuuint64_t dims[3] = {cuuint64_t(cols), cuuint64_t(rows), cuuint64_t(batch)}, strides[2] = {cuuint64_t(pitch) * 2, cuuint64_t(rows * pitch) * 2};
    const cuuint32_t box[3] = {32, 32, 1};
    return encode_tmap_bf16(map, p, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B);
}

template <int KIND, int SMS>
int launch_product(const Maps& maps, Args g, const DeviceInfo& dev, cudaStream_t s) {
    const auto kern = SMS == 2 ? pair_kernel<KIND> : single_kernel<KIND>;
    static bool configured[64] = {};
    if (!configured[dev.device & 63]) {
        MIMK_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<KIND>::SMEM));
        configured[dev.device & 63] = true;
    }
    g.tiles_m = int((g.rows + BM * SMS - 1) / (BM * SMS)), g.tiles_n = int((g.cols + BM * SMS - 1) / (BM * SMS));
    const int64_t per   = KIND == APPLY ? int64_t(g.tiles_m) * g.tiles_n : int64_t(g.tiles_m) * (g.tiles_m + 1) / 2, tiles = per * g.batch * g.splits;
    if (tiles >= (int64_t(1) << 30)) return MIMK_E_UNSUPPORTED;
    const int64_t most = dev.sm_count / SMS;
    return launch_after(kern, unsigned(SMS * (tiles < most ? tiles : most)), THREADS, Shape<KIND>::SMEM, s, maps, g);
}
// How a product runs: a tile on pairs of SMs or on single ones, and over how many tiles the k-blocks of one are dealt out; whichever ends first, in cycles. Measured: a
// k-block takes 540 cycles on a pair (256 x 256, of which the tensor cores need 512) and 500 on a single SM, whose 128 x 128 would be done in 256, had the 64 bytes a cycle that an SM gets
// from the L2 cache not to carry its operands; what a tile has at its ends some 6000; adding up partial results another launch of 12000 and their bytes.
struct How {
    int sms, splits, per, asked;
    double time;
};
How how(int kind, int64_t rows, int64_t cols, int64_t batch, int64_t kb, int sm_count, int least_splits, int most_splits) {
    How best{1, 1, int(kb), 1, 1e300};
    for (int sms = 1; sms <= 2; ++sms) {
        const int64_t m = (rows + BM * sms - 1) / (BM * sms), n = (cols + BM * sms - 1) / (BM * sms), tiles = (kind == APPLY ? m * n : m * (m + 1) / 2) * batch;
        for (int64_t splits = least_splits; splits <= most_splits; splits *= 2) {
            const int64_t per = (kb + splits - 1) / splits, rounds = (tiles * splits + sm_count / sms - 1) / (sm_count / sms);
            double time = double(rounds) * double(per) * (sms == 2 ? 540 : 500) + 6000.0 * double(rounds < 2 ? rounds : 2);
            if (splits > 1) time += 12000 + double(splits) * double(rows) * double(rows) * double(batch) * 4 / 3000;
            if (time < best.time) best = {sms, int((kb + per - 1) / per), int(per), int(splits), time};
        }
    }
    return best;
}
template <int KIND>
int launch(const Maps& maps, Args g, const How& h, const DeviceInfo& dev, cudaStream_t s) {
    g.splits = h.splits, g.per = h.per;
    MIMK_TRY((h.sms == 2 ? launch_product<KIND, 2>(maps, g, dev, s) : launch_product<KIND, 1>(maps, g, dev, s)));
    if (h.splits == 1) return MIMK_OK;
    const int64_t units = int64_t((g.rows + 7) / 8) * ((g.cols + 31) / 32) * g.batch;
    return launch_after(sum_kernel, unsigned((units + 7) / 8 < 65536 ? (units + 7) / 8 : 65536), 256, 0, s, g, h.splits);
}

template <class T>
int prepare(const Desc& d, const Plan& p, int64_t first, int64_t count, cudaStream_t s) {
    static thread_local Matrices all;
    bool vec = d.n % 8 == 0;
    for (int64_t i = 0; i < count; ++i) {
        all.x[i] = d.x[first + i];
        vec      = vec && aligned16(d.x[first + i]);
    }
    const int64_t values = d.m * d.n;
    const dim3 squares(unsigned(p.chunks), unsigned(count)), rows(unsigned(d.m < 4096 ? d.m : 4096), unsigned(count));
    if (vec) {
        MIMK_TRY(launch_after(squares_kernel<T, 8>, squares, PREPARE, 0, s, all, values, p.sums));
        return launch_after(prepare_kernel<T, 8>, rows, PREPARE, 0, s, all, int(d.m), int(d.n), int(p.pitch_x), static_cast<const double*>(p.sums), d.eps, p.x[0][0], p.x[0][1]);
    }
    MIMK_TRY(launch_after(squares_kernel<T, 1>, squares, PREPARE, 0, s, all, values, p.sums));
    return launch_after(prepare_kernel<T, 1>, rows, PREPARE, 0, s, all, int(d.m), int(d.n), int(p.pitch_x), static_cast<const double*>(p.sums), d.eps, p.x[0][0], p.x[0][1]);
}

// Matrices that a CTA takes whole.
bool small(const Desc& d) { return (d.m < d.n ? d.m : d.n) <= SMALL_K && (d.m < d.n ? d.n : d.m) <= SMALL_L; }
template <class T, bool TALL>
int small_launch(const Matrices& all, const SmallArgs& g, int64_t count, const DeviceInfo& dev, cudaStream_t s) {
    const auto kern = small_kernel<T, TALL>;
    static bool configured[64] = {};
    if (!configured[dev.device & 63]) {
        MIMK_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (2 * SMALL_L / 64 + 2) * CHUNK64 + 1024));
        configured[dev.device & 63] = true;
    }
    return launch_after(kern, unsigned(count), SMALL_THREADS, size_t(2 * g.chunks + 2) * CHUNK64 + 1024, s, all, g);
}
int small_all(const Desc& d, const Factors* f, const DeviceInfo& dev, cudaStream_t s) {
    static thread_local Matrices all;
    const bool tall = d.m > d.n;
    SmallArgs g;
    g.k = int(tall ? d.n : d.m), g.l = int(tall ? d.m : d.n), g.chunks = (g.l + 63) / 64, g.steps = d.steps, g.eps = d.eps, g.scale = d.scale, g.status = dev.status_dev;
    for (int i = 0; i < d.steps; ++i) g.f[i] = f[i];
    for (int64_t first = 0; first < d.batch; first += TABLE) {
        const int64_t count = d.batch - first < TABLE ? d.batch - first : TABLE;
        g.out = static_cast<__nv_bfloat16*>(d.out) + first * d.m * d.n;
        g.vec = d.n % 8 == 0 && aligned16(g.out);
        for (int64_t i = 0; i < count; ++i) all.x[i] = d.x[first + i], g.vec = g.vec && aligned16(d.x[first + i]);
        if (d.dtype == MIMK_F32) MIMK_TRY((tall ? small_launch<float, true>(all, g, count, dev, s) : small_launch<float, false>(all, g, count, dev, s)));
        else MIMK_TRY((tall ? small_launch<__nv_bfloat16, true>(all, g, count, dev, s) : small_launch<__nv_bfloat16, false>(all, g, count, dev, s)));
    }
    return MIMK_OK;
}

int slice(const Desc& d, const Plan& p, const Factors* f, int64_t first, int64_t count, const DeviceInfo& dev, cudaStream_t s) {
    MIMK_TRY(d.dtype == MIMK_F32 ? prepare<float>(d, p, first, count, s) : prepare<__nv_bfloat16>(d, p, first, count, s));
    const bool tall = d.m > d.n;
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(d.out) + first * d.m * d.n;
    const bool staged  = !group::tma_can_read(out, d.n);
    // Every map once, over all of a kind of buffers: the four of X (a first and a second f16, of one step and of the next) as an operand of each product and as tiles, A and B,
    // and the result's tiles. (Two microseconds of host time each.)
    CUtensorMap gram, apply, tiles, a_b, result;
    MIMK_TRY(map_of(&gram, p.x[0][0], d.m, d.n, p.pitch_x, 4 * p.slice, tall ? 64 : BM));
    MIMK_TRY(map_of(&apply, p.x[0][0], d.m, d.n, p.pitch_x, 4 * p.slice, tall ? BM : 64));
    MIMK_TRY(tile_map(&tiles, p.x[0][0], d.m, d.n, p.pitch_x, 4 * p.slice));
    MIMK_TRY(map_of(&a_b, p.a, p.k, p.k, p.pitch_a, 2 * p.slice, BM));
    MIMK_TRY(staged ? tile_map(&result, p.out, d.m, d.n, p.pitch_x, count) : tile_map(&result, out, d.m, d.n, d.n, count));
    const int z = int(p.slice);
    const int64_t kb_gram = ((tall ? d.m : d.n) + BK - 1) / BK, kb = (p.k + BK - 1) / BK;
    // (sums are split as for one matrix alone, so that it comes out the same in any batch)
    const int splits  = how(GRAM, p.k, p.k, 1, kb_gram, dev.sm_count, 1, p.splits).asked;
    const How hows[3] = {how(GRAM, p.k, p.k, count, kb_gram, dev.sm_count, splits, splits), how(SQUARE, p.k, p.k, count, kb, dev.sm_count, 1, 1), how(APPLY, d.m, d.n, count, kb, dev.sm_count, 1, 1)};
    Maps maps;
    for (int step = 0; step < d.steps; ++step) {
        const Factors& c = f[step];
        const int now = step & 1, next = now ^ 1;
        Args g{};
        g.batch = int(count), g.pitch = int(p.pitch_a), g.diag_pitch = int(p.pitch_d), g.status = dev.status_dev;
        // A
        g.rows = g.cols = int(p.k), g.kb = int(kb_gram), g.a_mn = g.b_mn = tall, g.out = p.a, g.diag_out = p.d, g.part = p.part;
        g.f[0] = 1.f / (SX * SX), g.f[4] = c.a;
        maps.left = maps.right = gram, g.z_left = g.z_right = 2 * now * z;
        MIMK_TRY(launch<GRAM>(maps, g, hows[0], dev, s));
        // B
        g.kb = int(kb), g.a_mn = g.b_mn = 0, g.in = p.a, g.out = p.b, g.diag_in = p.d, g.diag_out = p.e;
        g.f[0] = 1.f / (c.a * c.a), g.f[1] = 1.f / c.a, g.f[2] = c.q, g.f[3] = c.r, g.f[4] = c.b;
        maps.left = maps.right = a_b, g.z_left = g.z_right = 0;
        MIMK_TRY(launch<SQUARE>(maps, g, hows[1], dev, s));
        // X
        g.rows = int(d.m), g.cols = int(d.n), g.b_mn = !tall, g.tall = tall, g.last = step + 1 == d.steps, g.diag_in = p.e;
        g.f[0] = c.p, g.f[1] = 1.f / c.b, g.f[2] = d.scale / SX, g.f[3] = c.low;
        (tall ? maps.left : maps.right) = apply, (tall ? g.z_left : g.z_right) = 2 * now * z;
        (tall ? maps.right : maps.left) = a_b, (tall ? g.z_right : g.z_left) = z;
        maps.tile = tiles, g.z_hi = 2 * now * z, g.z_lo = g.z_hi + z;
        maps.out = g.last ? result : tiles, g.z_out_hi = g.last ? 0 : 2 * next * z, g.z_out_lo = g.z_out_hi + z;
        MIMK_TRY(launch<APPLY>(maps, g, hows[2], dev, s));
    }
    return staged ? copy_rows(p.out, p.pitch_x, out, d.n, count * d.m, d.n, s) : MIMK_OK;
}

}  // namespace
}  // namespace mimk

using namespace mimk;

extern "C" int mimk_orthogonalize_workspace(const mimk_orthogonalize_desc* d, uint64_t* bytes) {
    MIMK_TRY(check(d));
    if (!bytes) return MIMK_E_ARG;
    Space space(nullptr);
    if (!nothing(*d) && !small(*d)) plan(*d, space);
    *bytes = space.used();
    return MIMK_OK;
}

extern "C" int mimk_orthogonalize(const mimk_orthogonalize_desc* d, void* stream) {
    MIMK_TRY(check(d));
    Factors f[MOST_STEPS];
    MIMK_TRY(factors_of(*d, f));
    int st                = MIMK_OK;
    const DeviceInfo* dev = device_info(&st);
    if (!dev) return st;
    if (nothing(*d)) return MIMK_OK;
    if (!d->out) return MIMK_E_ARG;
    const size_t size = dtype_size(d->dtype);
    if (reinterpret_cast<uintptr_t>(d->out) % 2) return MIMK_E_ALIGN;
    for (int64_t i = 0; i < d->batch; ++i) {
        if (!d->x[i]) return MIMK_E_ARG;
        if (reinterpret_cast<uintptr_t>(d->x[i]) % size) return MIMK_E_ALIGN;
    }
    if (small(*d)) return small_all(*d, f, *dev, static_cast<cudaStream_t>(stream));
    Space space(d->workspace);
    const Plan p = plan(*d, space);
    if (!d->workspace || space.used() > d->workspace_bytes) return MIMK_E_WORKSPACE;
    if (!aligned16(d->workspace)) return MIMK_E_ALIGN;
    for (int64_t first = 0; first < d->batch; first += p.slice)
        MIMK_TRY(slice(*d, p, f, first, d->batch - first < p.slice ? d->batch - first : p.slice, *dev, static_cast<cudaStream_t>(stream)));
    return MIMK_OK;
}
