// Products of a training step on paired SMs: the pipeline of gemm_tc2.cu (TMA loads, one issuer of tcgen05.mma.cta_group::2, two accumulators in
// tensor memory and an epilogue that empties one while the other fills; here a warp for each operand's loads, and four or eight for the
// epilogue) with what gradients need beyond a forward product:
//   - either operand K-major or MN-major, so that x^T dy reads both matrices where the forward pass left them;
//   - two operand pairs added in one accumulator (da W1^T + db W3^T);
//   - several products in one launch (the three weight gradients and the input's), so that the last, half empty round of tiles comes once;
//   - the k-blocks of a tile dealt out over several tiles, each with an f32 partial result of its own, where there are few tiles;
//   - extents that are known on the device only (the rows that are left once those without a target are taken out);
//   - epilogues that keep what a gradient needs, or turn an accumulator into one, without the product ever being written.
// A tile is 256 rows (128 per CTA) by 256 columns (128 + 128 of two right operands for the gated form): 512 cycles for a k-block of 64.
// What bounds it: the tensor cores, and over more than some ms the power limit. [8192, 14336] x [14336, 4096]: 0.81 M cycles, the multiplications' own
// number; 0.60 ms from idle (1.6 PFLOP/s). Few rows: the latency of the loads in flight.
#pragma once

#include "common.cuh"
#include "sm100_pair.cuh"

namespace mimk {
namespace group {

using namespace sm100;

enum Epilogue {
    STORE,      // the result as bf16, or as f32 (stored or added to what is there)
    GATED_FWD,  // two right operands: a, b -> a and b as f32, silu(a) b as bf16
    GATED_BWD,  // dh, with a and b read -> da = dh b silu'(a) and db = dh silu(a), as bf16
    CE_STATS,   // logits -> per row and 128 columns the maximum and the sum of exp(l - maximum), and the target's logit
    CE_EXP,     // the same, and exp(l - maximum) in 16 bits of its own (exp_code)
    CE_GRAD,    // logits -> g (exp(l - lse) - [column is the target]) as bf16
};

constexpr int BM = 128, BK = 64, BN = 256;
constexpr int ACC_COLS = 256;
constexpr int A_BYTES = BM * BK * 2, B_BYTES = 128 * BK * 2, STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int GROUP_M = 8;
constexpr int SLOT = 4096;  // a [32 rows x 128 bytes] tile of an epilogue warp
constexpr int MAX_PROBLEMS = 4;

template <int EPI>
struct Shape {
    static constexpr bool GATED = EPI == GATED_FWD;
    // The loss is f32, and the tensor cores cut sums off where f32 rounds: an error of some 2^-25 of the value for each 16 terms, always towards zero
    // (4096 of them: 1.2e-6 of the loss, 1.2e-5 of a logit whose terms have one sign). For the loss k-blocks are therefore summed in runs, which the epilogue adds up in registers: a quarter
    // the error at 4096, and no time, as an accumulator is read while the other one fills. That takes two warps for a row's 256 columns.
    // CE_GRAD sums its logits the same way, to the same bits: exp(l - lse) of an l rounded otherwise than those in lse is off by the difference
    // (4096 terms, a logit of 30: 3.6e-4, where 1 - p is 1e-10).
    static constexpr bool LOSS  = EPI == CE_STATS || EPI == CE_EXP || EPI == CE_GRAD;
    static constexpr int RUN    = LOSS ? 16 : 1 << 30;                      // k-blocks in one accumulator
    // of the epilogue: eight where two for a row's columns pay (STORE: results of few
    // k-blocks are bound by it; 64 rows through 4096 x 14336 and back, 318 us with four, 308 with eight)
    static constexpr int WARPS  = LOSS || EPI == STORE ? 8 : 4;
    // one warp for each operand's loads and one for the multiplications, then the epilogue's. Eight of those hold 128 accumulators a thread: they come
    // in whole groups of four, which pass registers on (168 a thread at launch, 3 x 168 = 56 + 2 x 224).
    static constexpr int FIRST   = LOSS ? 4 : 3;
    static constexpr int THREADS = (FIRST + WARPS) * 32;
    static constexpr int WIDTH  = GATED ? 128 : 256;                        // result columns of a tile
    static constexpr int SLOTS  = EPI == GATED_BWD ? 24 : EPI == GATED_FWD || EPI == STORE ? 16 : EPI == CE_STATS ? 0 : 8;  // of all epilogue warps
    static constexpr int STAGES = SLOTS == 24 ? 4 : SLOTS == 16 ? 5 : 6;
    static constexpr int SMEM   = STAGES * STAGE_BYTES + SLOTS * SLOT + 1024 + 256;
};

struct Problem {
    int M, N;
    int kb[2];             // k-blocks of 64 of the first and the second operand pair
    int a_mn, b_mn;        // operand stored with its M (N) axis contiguous
    int splits, rows_pad;  // the k-blocks dealt out over that many tiles; partial result s starts at row s * rows_pad
    int out_f32, add;      // STORE: f32 result; added to what is there
    const int* dyn_m;      // rows that there are, at most M; null: M
    const int* dyn_k;      // K of the first pair, at most 64 kb[0]; null: all of it
};
struct Maps {
    CUtensorMap a[MAX_PROBLEMS][2], b[MAX_PROBLEMS][2], out[MAX_PROBLEMS], extra[2];
};
struct Args {
    Problem p[MAX_PROBLEMS];
    int count;
    // CE_STATS, CE_GRAD
    const int* target;   // [rows] column of the whole matrix, or -1
    const float* lse;    // [rows]
    const float* scale;  // [rows]
    float2* part;        // [rows][tiles of columns]
    float* target_logit;  // [rows]
    int column0;          // first column of this piece
    int* status;
};
// (a kernel's parameters: 4 KiB at most)
static_assert(sizeof(Maps) + sizeof(Args) <= 4096, "too many parameters");

#ifdef __CUDACC__

struct Bars {
    uint64_t full[6], empty[6], acc_full[2], acc_empty[2], in[8];
    uint32_t tmem_base;
    int abort_flag;
};
static_assert(sizeof(Bars) <= 256, "barrier block too large");

// Walks a launch's tiles in rising order; what belongs to a problem is worked out when its first tile is met.
template <int WIDTH>
struct Tile {
    int prob, m, n;     // problem; row and column the pair's tile starts at
    int rows;           // rows that the problem has
    int kb0, kb1;       // k-blocks [kb0, kb1) of both pairs' kfirst + kb[1]
    int kfirst, split;  // k-blocks of the first pair

    __device__ __forceinline__ Tile() : prob(-1), begin_(0), end_(0) {}
    // the `index`-th tile; false: there is none
    __device__ __forceinline__ bool at(const Args& g, int index) {
        while (index >= end_) {
            if (++prob >= g.count) return false;
            const Problem& p = g.p[prob];
            rows             = p.dyn_m ? min(p.M, *p.dyn_m) : p.M;
            tiles_m_ = (rows + 2 * BM - 1) / (2 * BM), tiles_n_ = (p.N + WIDTH - 1) / WIDTH;
            kfirst = p.dyn_k ? min(p.kb[0], (*p.dyn_k + BK - 1) / BK) : p.kb[0];
            splits_ = p.splits, per_ = (kfirst + p.kb[1] + splits_ - 1) / splits_, all_ = kfirst + p.kb[1];
            begin_ = end_, end_ += tiles_m_ * tiles_n_ * splits_;
        }
        unsigned i = unsigned(index - begin_);
        split      = 0;
        if (splits_ > 1) split = int(i / unsigned(tiles_m_ * tiles_n_)), i -= unsigned(split * tiles_m_ * tiles_n_);
        const unsigned per_group = unsigned(GROUP_M * tiles_n_), group = i / per_group, in_group = i - group * per_group;
        const unsigned size = min(unsigned(tiles_m_) - group * GROUP_M, unsigned(GROUP_M));
        const unsigned column = size == GROUP_M ? in_group / GROUP_M : in_group / size;
        m   = int(group * GROUP_M + (in_group - column * size)) * 2 * BM;
        n   = int(column) * WIDTH;
        kb0 = min(all_, split * per_), kb1 = min(all_, kb0 + per_);
        return true;
    }

  private:
    int begin_, end_, tiles_m_, tiles_n_, splits_, per_, all_;
};

__device__ __forceinline__ void st_shared_v4(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// This lane's row of a 128-byte-swizzled slot: 32 f32, or 32 bf16 from 16-byte piece `piece0` on.
__device__ __forceinline__ void put_f32(uint32_t slot, int lane, const float (&v)[32]) {
#pragma unroll
    for (int i = 0; i < 32; i += 4)
        st_shared_v4(slot + lane * 128 + ((uint32_t(i >> 2) ^ uint32_t(lane & 7)) << 4), __float_as_uint(v[i]), __float_as_uint(v[i + 1]),
                     __float_as_uint(v[i + 2]), __float_as_uint(v[i + 3]));
}
__device__ __forceinline__ void put_bf16(uint32_t slot, int lane, int piece0, const float (&v)[32]) {
#pragma unroll
    for (int i = 0; i < 32; i += 8)
        st_shared_v4(slot + lane * 128 + ((uint32_t(piece0 + (i >> 3)) ^ uint32_t(lane & 7)) << 4), pack_bf16x2(v[i], v[i + 1]),
                     pack_bf16x2(v[i + 2], v[i + 3]), pack_bf16x2(v[i + 4], v[i + 5]), pack_bf16x2(v[i + 6], v[i + 7]));
}
__device__ __forceinline__ void get_f32(uint32_t slot, int lane, float (&v)[32]) {
#pragma unroll
    for (int i = 0; i < 32; i += 4)
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v[i]), "=f"(v[i + 1]), "=f"(v[i + 2]), "=f"(v[i + 3])
                     : "r"(slot + lane * 128 + ((uint32_t(i >> 2) ^ uint32_t(lane & 7)) << 4))
                     : "memory");
}
__device__ __forceinline__ void get_acc(uint32_t at, float (&v)[32], bool empty) {
    uint32_t r[32];
    tmem_ld_32x32(at, r);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = empty ? 0.f : __uint_as_float(r[i]);
}
// A parameter in a register: asked for again in every k-block, it is read from constant memory again.
__device__ __forceinline__ int held(int v) {
    asm volatile("" : "+r"(v));
    return v;
}
// A value from 0 to 1 in 16 bits: the low seven bits of an f32's exponent and nine of its fraction (the bits above are zero), rounded half up. Ten
// significant bits down to 2^-126, where f16 has eleven down to 2^-14 only and bf16 has eight.
__device__ __forceinline__ uint32_t exp_code(float v) { return (__float_as_uint(v) + 0x2000u) >> 14; }
__device__ __forceinline__ float exp_of(uint32_t code) { return __uint_as_float(code << 14); }
// 1 / (1 + exp(-a)): 0 where exp(-a) overflows
__device__ __forceinline__ float sigmoid(float a) { return __fdividef(1.f, 1.f + __expf(-a)); }

template <int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Shape<EPI>::THREADS, 1)
group_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args g) {
    using S = Shape<EPI>;
    constexpr int STAGES = S::STAGES, WIDTH = S::WIDTH;
    constexpr int BH = WIDTH / 2, BH_BYTES = BH * BK * 2;  // columns (of each right operand) staged by this CTA
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = smem_u32(smem_raw), tile_base = (raw_addr + 1023u) & ~1023u;
    Bars* bars = reinterpret_cast<Bars*>(smem_raw + (tile_base - raw_addr) + STAGES * STAGE_BYTES + S::SLOTS * SLOT);
    volatile int* abort_flag = &bars->abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(smem_u32(&bars->full[s]), 1);
            mbar_init(smem_u32(&bars->empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&bars->acc_full[b]), 1);
            mbar_init(smem_u32(&bars->acc_empty[b]), 2 * S::WARPS * 32);
        }
        for (int w = 0; w < 8; ++w) mbar_init(smem_u32(&bars->in[w]), 1);
        bars->abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(&bars->tmem_base), 512);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&bars->tmem_base);
    after_previous();

    Tile<WIDTH> t;
    if (warp < S::FIRST) {
      if constexpr (S::LOSS) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
      if (warp == 0 || warp == 2) {
        // ---------------- TMA producers (both CTAs): warp 0 the left operand, warp 2 the right one or ones ----------------
        // (one thread for both took longer over a k-block than the multiplication)
        if (lane == 0) {
            const bool left = warp == 0;
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            for (int tile = pair; ok && t.at(g, tile); tile += num_pairs) {
                const Problem& p = g.p[t.prob];
                const int mn = held(left ? p.a_mn : p.b_mn), first = left ? t.m + int(rank) * BM : t.n + int(rank) * BH;
                const uint32_t base = tile_base + (left ? 0 : A_BYTES);
                // the k-blocks of one operand pair after those of the other
                const auto run = [&](const CUtensorMap* map, const CUtensorMap* second, int k, int end) {
                    for (; k < end; k += BK) {
                        if (!(ok = mbar_wait(smem_u32(&bars->empty[stage]), phase ^ 1u, abort_flag))) break;
                        const uint32_t full_even = map_to_cta(smem_u32(&bars->full[stage]), 0), at = base + stage * STAGE_BYTES;
                        if (left && rank == 0) mbar_expect_tx(smem_u32(&bars->full[stage]), 2 * STAGE_BYTES);  // all four producers' bytes
                        if (!mn) {
                            tma_load_2d_pair(at, map, k, first, full_even);
                            if (second) tma_load_2d_pair(at + BH_BYTES, second, k, first, full_even);
                        } else if (second) {
                            tma_load_2d_pair(at, map, first, k, full_even);
                            tma_load_2d_pair(at + BH_BYTES, second, first, k, full_even);
                        } else {
                            tma_load_2d_pair(at, map, first, k, full_even);
                            tma_load_2d_pair(at + BK * 128, map, first + 64, k, full_even);
                        }
                        if (++stage == STAGES) stage = 0, phase ^= 1u;
                    }
                };
                const CUtensorMap* m = left ? maps.a[t.prob] : maps.b[t.prob];
                if (S::GATED && left) {
                    // (128 rows of one left operand)
                    run(m, nullptr, t.kb0 * BK, t.kb1 * BK);
                } else if (S::GATED) {
                    run(m, m + 1, t.kb0 * BK, t.kb1 * BK);
                } else {
                    run(m, nullptr, t.kb0 * BK, min(t.kb1, t.kfirst) * BK);
                    if (ok) run(m + 1, nullptr, max(t.kb0 - t.kfirst, 0) * BK, (t.kb1 - t.kfirst) * BK);
                }
            }
        }
      } else if (warp == 1) {
        // ---------------- MMA issuer (even CTA only) ----------------
        if (lane == 0 && rank == 0) {
            uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
            bool ok = true;
            const uint64_t high = smem_desc_sw128(0, 0, 1024);
            for (int tile = pair; ok && t.at(g, tile); tile += num_pairs) {
                const Problem& p     = g.p[t.prob];
                const uint32_t idesc = idesc_bf16_f32(2 * BM, BN, p.a_mn, p.b_mn);
                // a descriptor's low word is the address >> 4 with the leading offset >> 4 above it, its high word is the same for all
                const uint32_t a_step = p.a_mn ? 2048 >> 4 : 32 >> 4, b_step = p.b_mn ? 2048 >> 4 : 32 >> 4;
                const uint32_t a_low = (p.a_mn ? BK * 128 >> 4 : 1) << 16, b_low = ((p.b_mn ? BK * 128 >> 4 : 1) << 16) + (A_BYTES >> 4);
                int from = t.kb0;
                do {  // (once for a tile without k-blocks, whose accumulator is not read)
                    const int to = min(t.kb1, from + S::RUN);
                    if (!(ok = mbar_wait(smem_u32(&bars->acc_empty[acc]), acc_phase ^ 1u, abort_flag))) break;
                    tc_fence_after();
                    for (int kb = from; kb < to; ++kb) {
                        if (!(ok = mbar_wait(smem_u32(&bars->full[stage]), phase, abort_flag))) break;
                        tc_fence_after();
                        const uint32_t at = (tile_base + stage * STAGE_BYTES) >> 4;
#pragma unroll
                        for (int k = 0; k < BK / 16; ++k)
                            mma_f16_ss_pair(tmem_base + acc * ACC_COLS, high | (at + a_low + k * a_step), high | (at + b_low + k * b_step), idesc,
                                            kb > from || k > 0);
                        mma_commit_pair(smem_u32(&bars->empty[stage]));
                        if (++stage == STAGES) stage = 0, phase ^= 1u;
                    }
                    if (!ok) break;
                    mma_commit_pair(smem_u32(&bars->acc_full[acc]));
                    if (++acc == 2) acc = 0, acc_phase ^= 1u;
                    from = to;
                } while (from < t.kb1);
            }
        }
      }
    } else {
        if constexpr (S::LOSS) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        // ---------------- epilogue (both CTAs): 32 rows for each warp (for each two of them, where there are eight), one per lane ----------------
        const int quarter = warp & 3;
        const uint32_t slots = tile_base + STAGES * STAGE_BYTES + (warp - S::FIRST) * (S::SLOTS / S::WARPS) * SLOT;
        const uint32_t in_bar = smem_u32(&bars->in[quarter * 2]);
        uint32_t acc = 0, acc_phase = 0, turn = 0, in_phase = 0;
        bool ok = true;
        bool have = t.at(g, pair);
        // GATED_BWD: a and b of 32 columns, two such pairs of slots in turn, requested as soon as a pair is free
        auto request = [&](const Tile<WIDTH>& at, int c) {
            if constexpr (EPI == GATED_BWD) {
                const int row = at.m + int(rank) * BM + quarter * 32, second = c >> 5 & 1;
                if (lane == 0 && row < at.rows && c < WIDTH && at.n + c < g.p[at.prob].N) {
                    mbar_expect_tx(in_bar + second * 8, 2 * SLOT);
                    tma_load_2d(slots + second * 2 * SLOT, &maps.extra[0], at.n + c, row, in_bar + second * 8);
                    tma_load_2d(slots + (second * 2 + 1) * SLOT, &maps.extra[1], at.n + c, row, in_bar + second * 8);
                }
            }
        };
        if (have) request(t, 0), request(t, 32);
        for (int tile = pair; have && ok;) {
            const Problem& p = g.p[t.prob];
            const int row0 = t.m + int(rank) * BM + quarter * 32, row = row0 + lane;
            // (products over rows read whole k-blocks of them: CE_GRAD writes zeros up to the end of the last one)
            const bool empty = t.kb0 == t.kb1, there = row0 < (EPI == CE_GRAD ? (t.rows + BK - 1) / BK * BK : t.rows);
            const int n0 = t.n, width = min(WIDTH, p.N - n0);  // (what lies past the last column is not worked on)
            uint32_t t0, acc_empty_even;
            auto next_acc = [&] {
                const bool full = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars->acc_full[acc]), acc_phase, abort_flag));
                tc_fence_after();
                t0             = tmem_base + acc * ACC_COLS + (uint32_t(quarter * 32) << 16);
                acc_empty_even = map_to_cta(smem_u32(&bars->acc_empty[acc]), 0);
                if (++acc == 2) acc = 0, acc_phase ^= 1u;
                return full;
            };
            auto release = [&] {  // after the last read of this accumulator
                tc_fence_before();
                mbar_arrive_cluster(acc_empty_even);
            };
            if (!(ok = next_acc())) break;
            // one slot's tile to a matrix, as a bulk group of its own (an empty one where the tile lies past the last column: a slot is free
            // by the number of groups committed since)
            auto send = [&](const CUtensorMap* m, uint32_t slot, int x, bool add = false, int down = 0) {
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    if (x < p.N) {
                        if (add) tma_reduce_add_2d(m, slot, x, row0 + down);
                        else tma_store_2d(m, slot, x, row0 + down);
                    }
                    bulk_commit();
                }
            };
            if (!there) {
                release();
                for (int kb = t.kb0 + min(S::RUN, t.kb1 - t.kb0); ok && kb < t.kb1; kb += S::RUN) {  // the tile's other accumulators
                    if ((ok = next_acc())) release();
                }
                if (!ok) break;
            } else if constexpr (EPI == STORE) {
                const int step = p.out_f32 ? 32 : 64, half = (warp - S::FIRST) >> 2 << 7, end = min(half + 128, width);
                if (half >= end) release();
#pragma unroll 1
                for (int c0 = half; c0 < end; c0 += step, ++turn) {
                    const uint32_t slot = slots + (turn & 1u) * SLOT;
                    if (lane == 0) bulk_wait_read_1();
                    __syncwarp();
                    float v[32];
                    get_acc(t0 + c0, v, empty);
                    if (p.out_f32) {
                        if (c0 + 32 >= end) release();
                        put_f32(slot, lane, v);
                    } else {
                        put_bf16(slot, lane, 0, v);
                        get_acc(t0 + c0 + 32, v, empty);
                        if (c0 + 64 >= end) release();
                        put_bf16(slot, lane, 4, v);
                    }
                    send(&maps.out[t.prob], slot, n0 + c0, p.add, t.split * p.rows_pad);
                }
            } else if constexpr (EPI == GATED_FWD) {
                // the accumulator's columns: [a | b] of the even CTA's columns, then [a | b] of the odd one's
#pragma unroll 1
                for (int c = 0; c < width; c += 32) {
                    const int ac = (c / BH) * 2 * BH + c % BH;
                    float a[32], b[32];
                    get_acc(t0 + ac, a, empty);
                    get_acc(t0 + ac + BH, b, empty);
                    if (c + 32 >= width) release();
                    // slots: a, b, h, h; whichever is next was last sent at least two groups ago
                    if (lane == 0) bulk_wait_read_1();
                    __syncwarp();
                    put_f32(slots, lane, a);
                    send(&maps.extra[0], slots, n0 + c);
                    if (lane == 0) bulk_wait_read_1();
                    __syncwarp();
                    put_f32(slots + SLOT, lane, b);
                    send(&maps.extra[1], slots + SLOT, n0 + c);
#pragma unroll
                    for (int i = 0; i < 32; ++i) a[i] = a[i] * sigmoid(a[i]) * b[i];
                    const uint32_t slot = slots + (2 + (turn & 1u)) * SLOT;
                    put_bf16(slot, lane, (c & 32) ? 4 : 0, a);
                    if ((c & 32) || c + 32 >= width) {
                        send(&maps.out[t.prob], slot, n0 + (c & ~63));
                        ++turn;
                    }
                }
            } else if constexpr (EPI == GATED_BWD) {
#pragma unroll 1
                for (int c = 0; c < width; c += 32) {
                    float a[32], b[32], d[32];
                    const uint32_t second = c >> 5 & 1, in = slots + second * 2 * SLOT;
                    if (!(ok = __all_sync(0xffffffffu, mbar_wait(in_bar + second * 8, in_phase >> second & 1u, abort_flag)))) break;
                    in_phase ^= 1u << second;
                    get_f32(in, lane, a);
                    get_f32(in + SLOT, lane, b);
                    __syncwarp();
                    request(t, c + 64);
                    get_acc(t0 + c, d, empty);
                    if (c + 32 >= width) release();
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float e = sigmoid(a[i]), gate = a[i] * e, db = d[i] * gate;
                        a[i] = d[i] * b[i] * (e + gate * (1.f - e));
                        b[i] = db;
                    }
                    if (!second) {
                        if (lane == 0) bulk_wait_read_0();
                        __syncwarp();
                    }
                    put_bf16(slots + 4 * SLOT, lane, second * 4, a);
                    put_bf16(slots + 5 * SLOT, lane, second * 4, b);
                    if (second || c + 32 >= width) {
                        send(&maps.out[0], slots + 4 * SLOT, n0 + (c & ~63));
                        send(&maps.out[1], slots + 5 * SLOT, n0 + (c & ~63));
                    }
                }
                if (!ok) break;
            } else if constexpr (S::LOSS) {
                // this warp's 128 of the columns, in registers: the runs of k-blocks added up
                const int half = (warp - S::FIRST) >> 2 << 7, n1 = n0 + half, left = p.N - n1;
                const int tcol = row < t.rows ? g.target[row] - g.column0 - n1 : -1;
                uint32_t raw[128];
#pragma unroll
                for (int c = 0; c < 128; c += 32) tmem_ld_32x32(t0 + half + c, *reinterpret_cast<uint32_t(*)[32]>(raw + c));
                tmem_ld_wait();
                release();
#pragma unroll 1
                for (int kb = t.kb0 + S::RUN; kb < t.kb1; kb += S::RUN) {
                    if (!(ok = next_acc())) break;
#pragma unroll
                    for (int c = 0; c < 128; c += 16) {
                        uint32_t r[16];
                        tmem_ld_32x16(t0 + half + c, r);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; ++i) raw[c + i] = __float_as_uint(__uint_as_float(raw[c + i]) + __uint_as_float(r[i]));
                    }
                    release();
                }
                if (!ok) break;
                float v[128];
#pragma unroll
                for (int i = 0; i < 128; ++i) v[i] = __uint_as_float(raw[i]);
                if constexpr (EPI == CE_GRAD) {
                    const bool mine = row < t.rows;
                    const float lse = mine ? g.lse[row] : 0.f, scale = mine ? g.scale[row] : 0.f;
                    // rows past the last one are zeros, which the products over rows read
#pragma unroll
                    for (int i = 0; i < 128; ++i) v[i] = mine ? scale * (__expf(v[i] - lse) - (tcol == i ? 1.f : 0.f)) : 0.f;
#pragma unroll
                    for (int c = 0; c < 128; c += 64) {
                        if (lane == 0) bulk_wait_read_0();
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 64; i += 8)
                            st_shared_v4(slots + lane * 128 + ((uint32_t(i >> 3) ^ uint32_t(lane & 7)) << 4), pack_bf16x2(v[c + i], v[c + i + 1]), pack_bf16x2(v[c + i + 2], v[c + i + 3]),
                                         pack_bf16x2(v[c + i + 4], v[c + i + 5]), pack_bf16x2(v[c + i + 6], v[c + i + 7]));
                        send(&maps.out[0], slots, n1 + c);
                    }
                } else {
                    if (left < 128) {
#pragma unroll
                        for (int i = 0; i < 128; ++i) v[i] = i < left ? v[i] : -INFINITY;
                    }
                    if (__any_sync(0xffffffffu, tcol >= 0 && tcol < 128)) {
#pragma unroll
                        for (int i = 0; i < 128; ++i)
                            if (tcol == i) g.target_logit[row] = v[i];
                    }
                    float top = -INFINITY, sum = 0.f;
#pragma unroll
                    for (int i = 0; i < 128; ++i) top = fmaxf(top, v[i]);
                    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
                    for (int c = 0; c < 128; c += 32) {
                        float part = 0.f;
#pragma unroll
                        for (int i = c; i < c + 32; ++i) v[i] = __expf(v[i] - base), part += v[i];
                        sum += part;
                    }
                    if (row < t.rows) g.part[int64_t(row) * ((p.N + 255) / 256 * 2) + (n1 >> 7)] = make_float2(top, sum);
                    if constexpr (EPI == CE_EXP) {
#pragma unroll
                        for (int c = 0; c < 128; c += 64) {
                            if (lane == 0) bulk_wait_read_0();
                            __syncwarp();
#pragma unroll
                            for (int i = 0; i < 64; i += 8)
                                st_shared_v4(slots + lane * 128 + ((uint32_t(i >> 3) ^ uint32_t(lane & 7)) << 4), __byte_perm(exp_code(v[c + i]), exp_code(v[c + i + 1]), 0x5410),
                                             __byte_perm(exp_code(v[c + i + 2]), exp_code(v[c + i + 3]), 0x5410), __byte_perm(exp_code(v[c + i + 4]), exp_code(v[c + i + 5]), 0x5410), __byte_perm(exp_code(v[c + i + 6]), exp_code(v[c + i + 7]), 0x5410));
                            send(&maps.out[0], slots, n1 + c);
                        }
                    }
                }
            }
            tile += num_pairs;
            have = t.at(g, tile);
            if (have) request(t, 0), request(t, 32);
        }
        if (lane == 0) bulk_wait_all();
    }

    // Neither CTA may release shared or tensor memory while the other can still touch it: meet first.
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 512);
    }
    if (threadIdx.x == 0 && *abort_flag) *g.status = MIMK_E_DEVICE_WAIT;
}

#endif

// ---- host ------------------------------------------------------------------------------------------------------------------------
// A row-major bf16 matrix whose rows are `pitch` elements apart.
struct Mat {
    const void* p;
    int64_t rows, cols, pitch;
};
inline bool tma_can_read(const void* p, int64_t pitch, int size = 2) { return aligned16(p) && (pitch * size) % 16 == 0; }

// The operand's map: `mn`: the matrix is [K, M or N], else [M or N, K]; `staged`: M or N values that a CTA stages.
inline int operand_map(CUtensorMap* map, const Mat& x, bool mn, int staged) {
    return make_tmap_2d(map, false, x.p, uint64_t(x.cols), uint64_t(x.rows), uint64_t(x.pitch) * 2, 64, mn ? 64u : uint32_t(staged));
}
inline int result_map(CUtensorMap* map, void* p, bool f32, int64_t rows, int64_t cols, int64_t pitch) {
    return make_tmap_2d(map, f32, p, uint64_t(cols), uint64_t(rows), uint64_t(pitch) * (f32 ? 4 : 2), f32 ? 32 : 64, 32);
}

template <int EPI>
int launch_group(const Maps& maps, const Args& args, const DeviceInfo& dev, cudaStream_t s) {
    auto kern = group_kernel<EPI>;
    static bool configured[64] = {};
    if (!configured[dev.device & 63]) {
        MIMK_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<EPI>::SMEM));
        configured[dev.device & 63] = true;
    }
    int64_t tiles = 0;
    for (int q = 0; q < args.count; ++q) {
        const Problem& p = args.p[q];
        tiles += int64_t((p.M + 2 * BM - 1) / (2 * BM)) * ((p.N + Shape<EPI>::WIDTH - 1) / Shape<EPI>::WIDTH) * p.splits;
    }
    if (tiles > (1 << 30)) return MIMK_E_UNSUPPORTED;
    const int64_t pairs = dev.sm_count / 2;
    const int grid      = int(2 * (tiles < pairs ? tiles : pairs));
    if (!grid) return MIMK_OK;
    return launch_after(kern, unsigned(grid), Shape<EPI>::THREADS, Shape<EPI>::SMEM, s, maps, args);
}

}  // namespace group
}  // namespace mimk
