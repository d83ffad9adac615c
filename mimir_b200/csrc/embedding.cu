// Token embedding and its gradient:  out[i] = scale table[ids[i]],   dtable[c] = scale sum over ids[i] = c of dy[i].
//
// The first is a copy of rows. For the second the positions are put in groups by class, without a sort: counted per class with integer atomics, a place
// for each class's group taken from a cursor, each position written to its group. Atomics leave a group's positions in any order, but their
// set is known, so each group is put in rising order before it is summed (32 positions by a warp, in registers; more of them by a block, as a map of
// bits), and results are the same call after call. A warp then owns 32 x VEC x COLS columns of a class: it adds up to 32 rows of dy, or writes zeros;
// classes of more rows are taken by whole blocks, a run of the rows for each warp, joined in shared memory. All of it is one launch whose blocks meet between
// its phases (and one that clears the counts). Up to 2048 positions: a launch of blocks that each look through all of them for the classes that are their own.
// What bounds it: the bytes. 8192 rows of 4096 bf16: 18 us, 7.3 TB/s (some of it from L2); their gradient for 131072 classes, 1.07 GB of zeros and sums: 206 us, 5.5 TB/s,
// of which some 25 go by before the first zeros, until all classes are counted. 3001 x 2048 of 50021 classes, 217 MB: 61 us. 515 x 777 f32 of 10007: 18 us.
#include "elements.cuh"
#include "train_common.cuh"

namespace mimk {

namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int WORKERS = 512, BLOCK = WORKERS + 32;  // of the launch whose blocks meet (the fewer of them, the sooner), and a warp that writes zeros
constexpr int ZEROS = 4096;          // bytes of one bulk store
constexpr int LIGHT = 32;            // positions of a class that one warp adds up
constexpr int PIECE = 512;           // and that one block does
constexpr int WINDOW = 1 << 17;      // positions in one map of bits
constexpr int SORTED = 4096;         // positions that fit in its place
constexpr int WARP_SORTED = SORTED / (WORKERS / 32);  // and in a warp's part of it
constexpr int64_t LIM = int64_t(1) << 31;

struct Ids {
    const void* p;
    int64_t ignore, v;
    int wide, has_ignore;
};
enum { NO_TOKEN = -1, BAD = -2 };
// the class of a position, or one of the above
__device__ __forceinline__ int class_at(const Ids& ids, int64_t i) {
    const int64_t id = ids.wide ? static_cast<const int64_t*>(ids.p)[i] : int64_t(static_cast<const int32_t*>(ids.p)[i]);
    if (ids.has_ignore && id == ids.ignore) return NO_TOKEN;
    return id >= 0 && id < ids.v ? int(id) : BAD;
}

// COLS loads of VEC elements, 32 lanes side by side, are a part of a row: one warp's work. Where nothing changes, the bits are stored as they came (8192 x 4096 bf16: 25 us
// by way of f32, 18 so).
template <class T, class O, int VEC, int COLS>
__global__ void __launch_bounds__(THREADS) rows_kernel(const T* table, Ids ids, O* out, int64_t n, int64_t d, int shift, float scale, int* status) {
    after_previous();
    const int lane = threadIdx.x & 31;
    const int64_t units = n << shift;  // (as many parts to a row as the next power of two)
    for (int64_t u = int64_t(blockIdx.x) * WARPS + (threadIdx.x >> 5); u < units; u += int64_t(gridDim.x) * WARPS) {
        const int64_t i = u >> shift, from = (u - (i << shift)) * (32 * VEC * COLS) + lane * VEC;
        if (from - lane * VEC >= d) continue;
        const int c = class_at(ids, i);
        if (c == BAD && lane == 0) *status = MIMK_E_SHAPE;
        const int left = int(min(d - from, int64_t(32 * VEC * COLS)));  // (not above zero: this lane has none of the row)
        O* to          = out + i * d + from;
        if (c < 0) {
            float v[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = c == BAD ? NAN : 0.f;
#pragma unroll
            for (int k = 0; k < COLS; ++k)
                if (k * 32 * VEC < left) put(to + k * 32 * VEC, v);
            continue;
        }
        const T* row = table + int64_t(c) * d + from;
        Run<T, VEC> run[COLS];
#pragma unroll
        for (int k = 0; k < COLS; ++k)
            if (k * 32 * VEC < left) run[k].load(row + k * 32 * VEC);
        if constexpr (sizeof(T) == sizeof(O)) {
            if (scale == 1.f) {  // the values as they are
#pragma unroll
                for (int k = 0; k < COLS; ++k)
                    if (k * 32 * VEC < left) run[k].store(to + k * 32 * VEC);
                continue;
            }
        }
#pragma unroll
        for (int k = 0; k < COLS; ++k) {
            if (k * 32 * VEC >= left) break;
            float v[VEC];
            run[k].get(v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] *= scale;
            put(to + k * 32 * VEC, v);
        }
    }
}

template <int N>
__device__ __forceinline__ void workers_meet() {
    asm volatile("bar.sync 1, %0;" ::"n"(N) : "memory");
}
template <int N>
__device__ __forceinline__ void with_writer() {
    asm volatile("bar.sync 2, %0;" ::"n"(N) : "memory");
}

// ---- zeros -----------------------------------------------------------------------------------------------------------------------
// Bulk stores from a piece of shared memory that holds zeros, OUTSTANDING of them on their way. By themselves 32 KiB or so for each SM write 1.07 GB in 150 to 176 us, as stores by
// all threads do at best; beside the sums of 8192 rows stores of 2 KiB took 248 us (130 cycles each), of 4 KiB 208.
template <int OUTSTANDING>
__device__ __forceinline__ void zero_span(uint8_t* p, int64_t bytes, uint32_t zeros) {
    const int lane = threadIdx.x & 31;
    const int64_t head = min(bytes, int64_t(-reinterpret_cast<uintptr_t>(p) & 15)), body = (bytes - head) & ~int64_t(15), tail = bytes - head - body;
    // (elements are two or four bytes, on such boundaries)
    if (lane * 2 < head) *reinterpret_cast<uint16_t*>(p + lane * 2) = 0;
    if (lane * 2 < tail) *reinterpret_cast<uint16_t*>(p + head + body + lane * 2) = 0;
    if (lane == 0)
        for (int64_t at = 0; at < body; at += ZEROS) {
            asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(p + head + at), "r"(zeros), "r"(int(min(body - at, int64_t(ZEROS)))) : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(OUTSTANDING - 1) : "memory");
        }
}
__device__ __forceinline__ uint32_t make_zeros(uint4* room) {
    for (int i = threadIdx.x & 31; i < ZEROS / 16; i += 32) room[i] = make_uint4(0, 0, 0, 0);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    return uint32_t(__cvta_generic_to_shared(room));
}
__device__ __forceinline__ void zeros_written() {
    if ((threadIdx.x & 31) == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// ---- groups ------------------------------------------------------------------------------------------------------------------------
struct Groups {
    int* count;   // [v] positions of a class
    int* start;   // [v] where its group begins
    int* slot;    // [n] place in the group, in any order
    int* order;   // [n] positions by group
    int* sorted;  // [n] the same, groups of more than LIGHT positions in rising order
    int4* heavy;  // pieces of such groups: class, which piece, of how many, place of the partial sums where there are several
    int* light;   // [n] the other classes that occur
    int* whole;   // the classes of such groups: those of up to WARP_SORTED positions from the front, others from the end
    float* part;  // rows of partial sums
    int* cursor;  // places taken; pieces; blocks that have met; whether one gave up; the other classes; rows of partial sums; classes at the front and at the end of `whole`; of those put in order by blocks, how many are taken
    int64_t part_pitch, wholes;
};
constexpr int CURSORS = 9;

__global__ void __launch_bounds__(THREADS) clear_kernel(Groups g, int64_t v) {
    after_previous();
    if (blockIdx.x == 0 && threadIdx.x < CURSORS) g.cursor[threadIdx.x] = 0;
    for (int64_t i = int64_t(blockIdx.x) * THREADS + threadIdx.x; i < v; i += int64_t(gridDim.x) * THREADS) g.count[i] = 0;
}

// All blocks of the launch (which are resident at once) have come here. False: one of them has not come in a second or so (longer for many positions, whose phases take
// up to some cycles each where one class has most of them), the status word says so, and the kernel is left by all.
__device__ __forceinline__ bool all_blocks_meet(const Groups& g, int64_t n, int nth, int* status) {
    __shared__ int met;
    workers_meet<WORKERS>();
    if (threadIdx.x == 0) {
        int* arrived = g.cursor + 2;
        volatile int* given_up = g.cursor + 3;
        __threadfence();
        atomicAdd(arrived, 1);
        const int all      = nth * int(gridDim.x);
        const long long t0 = clock64();
        met = 1;
        for (;;) {
            int now;
            asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(now) : "l"(arrived) : "memory");
            if (now >= all) break;
            if (*given_up || clock64() - t0 > 2000000000LL + 16 * n) {
                *given_up = 1, *status = MIMK_E_DEVICE_WAIT, met = 0;
                break;
            }
        }
    }
    workers_meet<WORKERS>();
    return met;
}

__device__ __forceinline__ void count_positions(const Ids& ids, const Groups& g, int64_t n, int* status) {
    for (int64_t base = int64_t(blockIdx.x) * WORKERS; base < n; base += int64_t(gridDim.x) * WORKERS) {
        const int64_t i = base + threadIdx.x;
        const int c     = i < n ? class_at(ids, i) : NO_TOKEN;
        if (c == BAD) *status = MIMK_E_SHAPE;
        // one atomic for the lanes of one class
        const unsigned same = __match_any_sync(0xffffffffu, c), before = same & ((1u << (threadIdx.x & 31)) - 1);
        int first           = 0;
        if (!before && c >= 0) first = atomicAdd(g.count + c, __popc(same));
        first = __shfl_sync(0xffffffffu, first, __ffs(same) - 1);
        if (i < n) g.slot[i] = c >= 0 ? first + __popc(before) : -1;
    }
}

// the sum of a value over the threads of the block before this one, and over all
__device__ __forceinline__ int block_before(int v, int* total) {
    __shared__ int part[WORKERS / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int sum = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int w = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += w;
    }
    workers_meet<WORKERS>();  // (of an earlier call's reads)
    if (lane == 31) part[warp] = sum;
    workers_meet<WORKERS>();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < WORKERS / 32; ++w) {
        before += w < warp ? part[w] : 0;
        all += part[w];
    }
    *total = all;
    return before + sum - v;
}

__device__ __forceinline__ void take_places(const Groups& g, int64_t v) {
    __shared__ int first[6];
    for (int64_t base = int64_t(blockIdx.x) * WORKERS; base < v; base += int64_t(gridDim.x) * WORKERS) {
        const int64_t c = base + threadIdx.x;
        const int count = c < v ? g.count[c] : 0;
        const int pieces = count > LIGHT ? (count + PIECE - 1) / PIECE : 0, parts = pieces > 1 ? pieces : 0;
        int all, heavies, partials;
        const int before = block_before(count, &all);
        if (!all) continue;
        const int nth = block_before(pieces, &heavies), row = block_before(parts, &partials);
        // light classes, those for a warp and those for a block: ten bits each
        const bool light = count > 0 && !pieces, some = pieces && count <= WARP_SORTED, much = pieces && !some;
        int kinds;
        const int other = block_before(int(light) | int(some) << 10 | int(much) << 20, &kinds), lights = kinds & 1023, somes = kinds >> 10 & 1023, muches = kinds >> 20;
        if (threadIdx.x == 0) first[0] = atomicAdd(g.cursor, all);
        if (threadIdx.x == 32 && heavies) first[1] = atomicAdd(g.cursor + 1, heavies);
        if (threadIdx.x == 64 && lights) first[2] = atomicAdd(g.cursor + 4, lights);
        if (threadIdx.x == 96 && partials) first[3] = atomicAdd(g.cursor + 5, partials);
        if (threadIdx.x == 128 && somes) first[4] = atomicAdd(g.cursor + 6, somes);
        if (threadIdx.x == 160 && muches) first[5] = atomicAdd(g.cursor + 7, muches);
        workers_meet<WORKERS>();
        if (count) g.start[c] = first[0] + before;
        for (int k = 0; k < pieces; ++k) g.heavy[first[1] + nth + k] = make_int4(int(c), k, pieces, first[3] + row);
        if (light) g.light[first[2] + (other & 1023)] = int(c);
        if (some) g.whole[first[4] + (other >> 10 & 1023)] = int(c);
        if (much) g.whole[g.wholes - 1 - first[5] - (other >> 20)] = int(c);
        workers_meet<WORKERS>();
    }
}

__device__ __forceinline__ void fill_groups(const Ids& ids, const Groups& g, int64_t n) {
    for (int64_t i = int64_t(blockIdx.x) * WORKERS + threadIdx.x; i < n; i += int64_t(gridDim.x) * WORKERS) {
        const int slot = g.slot[i];
        if (slot >= 0) g.order[g.start[class_at(ids, i)] + slot] = int(i);
    }
}

// `size` values in shared memory, a power of two, in rising order (a bitonic network), by `threads` of which this is the t-th.
template <class Meet>
__device__ __forceinline__ void sort_shared(int* held, int size, int t, int threads, Meet&& meet) {
    for (int run = 2; run <= size; run *= 2)
        for (int step = run / 2; step; step /= 2) {
            for (int k = t; k < size / 2; k += threads) {
                const int at = 2 * k - (k & (step - 1)), a = held[at], b = held[at + step];
                if ((a > b) == ((at & run) == 0)) held[at] = b, held[at + step] = a;
            }
            meet();
        }
}
// The groups of heavy classes put in order. Where there are more of them than blocks, those of up to WARP_SORTED positions by a warp, in its part of the room. Others by a block, as bits of a map that are read off in order; where there
// are more positions than one map's, groups of up to SORTED in the map's place, and groups of more than a map's positions as the ids name them, which are fewer than the
// group over again for each map. (1048576 positions in 26214 classes, 64 columns of bf16: 681 us; 3531 with maps alone, 1099 with all sorted by blocks.)
// A block that is done takes the next group that nobody has, so that blocks end within one group's time of each other, however the classes follow one another: a few cycles for each of
// all positions at most, far below the limit of the meeting that follows. (22429696 positions in 148 classes: 19 ms; with a fixed share of the list of pieces one block had all of these, 2.1 s, and the others gave up.)
__device__ __forceinline__ void sort_heavies(const Ids& ids, const Groups& g, int64_t n, uint32_t* bits) {
    __shared__ int taken;
    const int some = g.cursor[6], much = g.cursor[7], warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool many = some + much > int(gridDim.x);
    for (int h = blockIdx.x + warp * gridDim.x; many && h < some; h += gridDim.x * (WORKERS / 32)) {
        const int c = g.whole[h], count = g.count[c], start = g.start[c];
        int* held = reinterpret_cast<int*>(bits) + warp * WARP_SORTED;
        int size  = 2 * LIGHT;
        while (size < count) size *= 2;
        for (int k = lane; k < size; k += 32) held[k] = k < count ? g.order[start + k] : INT_MAX;
        __syncwarp();
        sort_shared(held, size, lane, 32, [] { __syncwarp(); });
        for (int k = lane; k < count; k += 32) g.sorted[start + k] = held[k];
        __syncwarp();
    }
    const int groups   = much + (many ? 0 : some);
    const auto advance = [&] {
        workers_meet<WORKERS>();
        if (threadIdx.x == 0) taken = groups > int(gridDim.x) ? int(gridDim.x) + atomicAdd(g.cursor + 8, 1) : groups;
    };
    if (threadIdx.x == 0) taken = blockIdx.x;
    for (;; advance()) {
        workers_meet<WORKERS>();
        const int h = taken;
        if (h >= groups) break;
        const int c = h < much ? g.whole[g.wholes - 1 - h] : g.whole[h - much], count = g.count[c], start = g.start[c];
        if (n > WINDOW && count <= SORTED) {
            int* held = reinterpret_cast<int*>(bits);
            int size  = 2 * LIGHT;
            while (size < count) size *= 2;
            for (int k = threadIdx.x; k < size; k += WORKERS) held[k] = k < count ? g.order[start + k] : INT_MAX;
            workers_meet<WORKERS>();
            sort_shared(held, size, threadIdx.x, WORKERS, [] { workers_meet<WORKERS>(); });
            for (int k = threadIdx.x; k < count; k += WORKERS) g.sorted[start + k] = held[k];
            workers_meet<WORKERS>();
            continue;
        }
        int done = 0;
        if (count > WINDOW) {
            constexpr int EACH = 4;
            for (int64_t base = 0; base < n && done < count; base += WORKERS * EACH) {
                const int64_t first = base + threadIdx.x * EACH;
                unsigned its        = 0;
#pragma unroll
                for (int k = 0; k < EACH; ++k) its |= unsigned(first + k < n && class_at(ids, first + k) == c) << k;
                int all, to = start + done + block_before(__popc(its), &all);
                for (; its; its &= its - 1) g.sorted[to++] = int(first) + __ffs(its) - 1;
                done += all;
            }
            continue;
        }
        for (int64_t window = 0; window < n && done < count; window += WINDOW) {
            const int words = int(n - window < WINDOW ? (n - window + 31) / 32 : WINDOW / 32);
            const int each  = (words + WORKERS - 1) / WORKERS;
            for (int w = threadIdx.x; w < words; w += WORKERS) bits[w] = 0;
            workers_meet<WORKERS>();
            for (int k = threadIdx.x; k < count; k += WORKERS) {
                const int64_t at = g.order[start + k] - window;
                if (at >= 0 && at < WINDOW) atomicOr(bits + (at >> 5), 1u << (at & 31));
            }
            workers_meet<WORKERS>();
            const int lo = min(words, int(threadIdx.x) * each), hi = min(words, lo + each);
            int mine = 0, all;
            for (int w = lo; w < hi; ++w) mine += __popc(bits[w]);
            int to = start + done + block_before(mine, &all);
            for (int w = lo; w < hi; ++w)
                for (uint32_t b = bits[w]; b; b &= b - 1) g.sorted[to++] = int(window) + w * 32 + __ffs(b) - 1;
            done += all;
            workers_meet<WORKERS>();
        }
    }
}

// up to 32 values in rising order, one a lane (a bitonic network)
__device__ __forceinline__ int sorted_lanes(int v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int step = size >> 1; step; step >>= 1) {
            const int w     = __shfl_xor_sync(0xffffffffu, v, step);
            const bool less = ((lane & step) == 0) == ((lane & size) == 0);
            v = less ? min(v, w) : max(v, w);
        }
    return v;
}

// acc += the rows of dy at the positions that lanes 0 .. count - 1 hold, in that order, this lane's columns
template <class T, int VEC, int COLS>
__device__ __forceinline__ void add_rows(float (&acc)[COLS][VEC], const T* dy, int64_t d, int64_t from, int position, int count) {
    constexpr int AHEAD = 4;
    for (int k = 0; k < count; k += AHEAD) {
        Run<T, VEC> run[AHEAD][COLS];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            const int64_t row = __shfl_sync(0xffffffffu, position, min(k + a, 31));
#pragma unroll
            for (int q = 0; q < COLS; ++q) {
                const int64_t at = from + q * 32 * VEC;
                run[a][q].clear();
                if (k + a < count && at < d) run[a][q].load(dy + row * d + at);
            }
        }
#pragma unroll
        for (int a = 0; a < AHEAD; ++a)
#pragma unroll
            for (int q = 0; q < COLS; ++q) {
                float v[VEC];
                run[a][q].get(v);
                if (k + a < count)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) acc[q][j] += v[j];
            }
    }
}
template <class O, int VEC>
__device__ __forceinline__ void store_one(const float (&acc)[VEC], O* to, float scale, bool add) {
    float v[VEC], old[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) old[j] = 0.f;
    if (add) {
        Run<O, VEC> r;
        r.load(to), r.get(old);
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = add ? fmaf(acc[j], scale, old[j]) : acc[j] * scale;
    put(to, v);
}
template <class O, int VEC, int COLS>
__device__ __forceinline__ void store_row(const float (&acc)[COLS][VEC], O* row, int64_t d, int64_t from, float scale, bool add) {
#pragma unroll
    for (int q = 0; q < COLS; ++q) {
        const int64_t at = from + q * 32 * VEC;
        if (at < d) store_one<O, VEC>(acc[q], row + at, scale, add);
    }
}

// What the N workers' warps of a block have summed of one row's part, joined in their order and stored, 32 x VEC columns to a warp.
template <int N, class O, int VEC, int COLS>
__device__ __forceinline__ void join_warps(float (&acc)[COLS][VEC], float (*joined)[32 * VEC], O* row, int64_t d, int64_t from, float scale, bool add) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int q = 0; q < COLS; ++q) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) joined[warp][j * 32 + lane] = acc[q][j];
        workers_meet<N * 32>();
        const int64_t at = from + q * 32 * VEC;
        if (warp == q % N && at < d) {
            float all[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                all[j] = 0.f;
#pragma unroll 8
                for (int w = 0; w < N; ++w) all[j] += joined[w][j * 32 + lane];
            }
            store_one<O, VEC>(all, row + at, scale, add);
        }
        workers_meet<N * 32>();
    }
}

template <class T, class O, int VEC, int COLS>
__global__ void __launch_bounds__(BLOCK, 1) grad_kernel(const T* dy, Ids ids, Groups g, O* dtable, int64_t n, int64_t d, int64_t v, int shift, float scale, bool add, int* status) {
    constexpr int PART = 32 * VEC * COLS;
    __shared__ union {
        float joined[WORKERS / 32][32 * VEC];
        uint32_t bits[WINDOW / 32];
    } room;
    __shared__ alignas(16) uint4 nothing[ZEROS / 16];
    __shared__ int counted;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x >= WORKERS) {
        // the rows of classes that no position names, as soon as those are known: every gridDim.x-th 32 classes, neighbours among them together
        const uint32_t zeros = make_zeros(nothing);
        with_writer<BLOCK>();
        if (!counted || add) return;
        const int64_t row = d * int64_t(sizeof(O)), step = int64_t(gridDim.x) * 32, first = int64_t(blockIdx.x) * 32;
        int next = first + lane < v ? g.count[first + lane] : -1;
        for (int64_t base = first; base < v; base += step) {
            unsigned left = __ballot_sync(0xffffffffu, next == 0);
            next          = base + step + lane < v ? g.count[base + step + lane] : -1;
            while (left) {
                const int from = __ffs(left) - 1, to = min(32, from + (~(left >> from) ? __ffs(~(left >> from)) - 1 : 32));
                zero_span<8>(reinterpret_cast<uint8_t*>(dtable) + (base + from) * row, (to - from) * row, zeros);
                left = to == 32 ? 0u : left >> to << to;
            }
        }
        zeros_written();
        return;
    }
    // (launched together: the blocks meet)
    count_positions(ids, g, n, status);
    const bool met = all_blocks_meet(g, n, 1, status);
    if (threadIdx.x == 0) counted = met;
    with_writer<BLOCK>();
    if (!met) return;
    take_places(g, v);
    if (!all_blocks_meet(g, n, 2, status)) return;
    fill_groups(ids, g, n);
    if (!all_blocks_meet(g, n, 3, status)) return;
    if (g.cursor[1]) {
        sort_heavies(ids, g, n, room.bits);
        if (!all_blocks_meet(g, n, 4, status)) return;
    }
    const int64_t heavy_units = int64_t(g.cursor[1]) << shift;
    for (int64_t u = blockIdx.x; u < heavy_units; u += gridDim.x) {
        const int64_t h = u >> shift, first = (u - (h << shift)) * PART, from = first + lane * VEC;
        if (first >= d) continue;
        const int4 piece = g.heavy[h];
        const int c = piece.x, start = g.start[c] + piece.y * PIECE, count = min(PIECE, g.count[c] - piece.y * PIECE);
        const int each = (count + WORKERS / 32 - 1) / (WORKERS / 32), lo = min(count, warp * each), hi = min(count, lo + each);
        float acc[COLS][VEC] = {};
        for (int k = lo; k < hi; k += 32) add_rows<T, VEC, COLS>(acc, dy, d, from, k + lane < hi ? g.sorted[start + k + lane] : 0, min(32, hi - k));
        if (piece.z == 1) join_warps<WORKERS / 32, O, VEC, COLS>(acc, room.joined, dtable + int64_t(c) * d, d, from, scale, add);
        else join_warps<WORKERS / 32, float, VEC, COLS>(acc, room.joined, g.part + int64_t(piece.w + piece.y) * g.part_pitch, d, from, 1.f, false);
    }
    // The other classes that occur: units warp, warp + warps, ...; what 32 of them need to know comes in one load each, the positions of one while the rows of the one before
    // are on their way (a read takes several microseconds while zeros are written).
    const int64_t units = int64_t(g.cursor[4]) << shift, warps = int64_t(gridDim.x) * (WORKERS / 32);
    for (int64_t first = int64_t(warp) * gridDim.x + blockIdx.x; first < units; first += 32 * warps) {
        const int64_t mine = first + lane * warps;
        const int its      = mine < units ? g.light[mine >> shift] : 0;
        const int count = mine < units ? g.count[its] : 0, start = mine < units ? g.start[its] : 0;
        const int here  = int(min(int64_t(32), (units - first + warps - 1) / warps));
        const auto ask  = [&](int k) {
            const int positions = __shfl_sync(0xffffffffu, count, k & 31), begin = __shfl_sync(0xffffffffu, start, k & 31);
            return k < here && lane < positions ? g.order[begin + lane] : INT_MAX;
        };
        int next = ask(0);
        for (int k = 0; k < here; ++k) {
            const int position  = sorted_lanes(next), positions = __shfl_sync(0xffffffffu, count, k), c = __shfl_sync(0xffffffffu, its, k);
            const int64_t begin = ((first + k * warps) & ((int64_t(1) << shift) - 1)) * PART, from = begin + lane * VEC;
            next                = ask(k + 1);
            if (begin >= d) continue;
            float acc[COLS][VEC] = {};
            add_rows<T, VEC, COLS>(acc, dy, d, from, position, positions);
            store_row<O, VEC, COLS>(acc, dtable + int64_t(c) * d, d, from, scale, add);
        }
    }
    if (!g.cursor[5]) return;
    // what pieces of one class left, in their order
    if (!all_blocks_meet(g, n, 5, status)) return;
    for (int64_t u = int64_t(blockIdx.x) * (WORKERS / 32) + warp; u < heavy_units; u += warps) {
        const int64_t h = u >> shift, begin = (u - (h << shift)) * PART, from = begin + lane * VEC;
        const int4 piece = g.heavy[h];
        if (begin >= d || piece.y || piece.z == 1) continue;
        float acc[COLS][VEC] = {};
#pragma unroll
        for (int q = 0; q < COLS; ++q) {
            const int64_t at = from + q * 32 * VEC;
            if (at >= d) break;
            for (int k = 0; k < piece.z; ++k) {
                Run<float, VEC> run;
                float v[VEC];
                run.load(g.part + int64_t(piece.w + k) * g.part_pitch + at), run.get(v);
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[q][j] += v[j];
            }
        }
        store_row<O, VEC, COLS>(acc, dtable + int64_t(piece.x) * d, d, from, scale, add);
    }
}

// ---- few positions ---------------------------------------------------------------------------------------------------------------
// A block has every `group`-th class (blockIdx.x, blockIdx.x + groups, ...) and a part of the columns. Its warps look through a run of the positions each and
// list what belongs to those classes, in order; the classes that there are then take their positions off the lists.
constexpr int FEW = 2048, RUN = FEW / WARPS, OWN = 2048, AT_ONCE = 4;  // positions, of them a warp's, classes that a block counts at a time, positions that one warp adds up
template <class T, class O, int VEC, int COLS>
__global__ void __launch_bounds__(THREADS) few_kernel(const T* dy, Ids ids, O* dtable, int n, int64_t d, int v, int log_groups, float scale, bool add, int* status) {
    constexpr int PART = 32 * VEC * COLS;
    __shared__ int list[WARPS][RUN];          // position | local class << 11
    __shared__ int length[WARPS];
    __shared__ uint16_t counts[OWN];
    __shared__ uint16_t heavy[FEW / 5];       // local classes of more than AT_ONCE positions
    __shared__ int heavies;
    __shared__ float joined[WARPS][32 * VEC];
    after_previous();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, groups = 1 << log_groups, own = ((v - 1 - int(blockIdx.x)) >> log_groups) + 1;  // (no more groups than classes)
    const int64_t from = int64_t(blockIdx.y) * PART + lane * VEC;
    // (a window of the block's classes: all of them, unless there are more than 2048)
    for (int window = 0;; window += OWN) {
        const int here = min(OWN, own - window);
        for (int i = threadIdx.x; i < here; i += THREADS) counts[i] = 0;
        if (threadIdx.x == 0) heavies = 0;
        const int each = (n + WARPS - 1) / WARPS, begin = min(n, warp * each), end = min(n, begin + each);
        int found = 0;
        for (int base = begin; base < end; base += 32) {
            const int i = base + lane;
            const int c = i < end ? class_at(ids, i) : NO_TOKEN;
            if (c == BAD) *status = MIMK_E_SHAPE;
            const int local = (c >> log_groups) - window;
            const bool mine = c >= 0 && (c & (groups - 1)) == int(blockIdx.x) && local >= 0 && local < here;
            const unsigned all = __ballot_sync(0xffffffffu, mine);
            if (mine) list[warp][found + __popc(all & ((1u << lane) - 1))] = i | local << 11;
            found += __popc(all);
        }
        if (lane == 0) length[warp] = found;
        workers_meet<THREADS>();
        // how many each class has: a class's first position in its warp's list adds all of that list's
        for (int w = 0; w < WARPS; ++w) {
            if (warp == w)
                for (int base = 0; base < found; base += 32) {
                    const int local = base + lane < found ? list[w][base + lane] >> 11 : -1;
                    const unsigned same = __match_any_sync(0xffffffffu, local);
                    if (local >= 0 && __ffs(same) - 1 == lane) {
                        const int before = counts[local], now = before + __popc(same);
                        counts[local] = uint16_t(now);
                        if (before <= AT_ONCE && now > AT_ONCE) heavy[atomicAdd(&heavies, 1)] = uint16_t(local);
                    }
                    __syncwarp();
                }
            workers_meet<THREADS>();
        }
        // A class's positions in list w, behind the `held` that lanes hold: lane k takes the (k - held)-th of them.
        const auto take = [&](int w, int base, int local, int& position, int held) {
            const int entry    = base + lane < length[w] ? list[w][base + lane] : -1;
            const unsigned all = __ballot_sync(0xffffffffu, entry >= 0 && entry >> 11 == local);
            if (!all) return 0;
            const int nth = lane - held, source = nth >= 0 && nth < __popc(all) ? int(__fns(all, 0, nth + 1)) : 0;
            const int its = __shfl_sync(0xffffffffu, entry, source);
            if (nth >= 0 && nth < __popc(all)) position = its & (FEW - 1);
            return __popc(all);
        };
        // classes of several positions (each by itself: in whichever order): by the block, a list to a warp
        for (int h = 0; h < heavies; ++h) {
            const int local = heavy[h];
            float acc[COLS][VEC] = {};
            for (int base = 0; base < length[warp]; base += 32) {
                int position = 0;
                if (const int count = take(warp, base, local, position, 0)) add_rows<T, VEC, COLS>(acc, dy, d, from, position, count);
            }
            join_warps<WARPS, O, VEC, COLS>(acc, joined, dtable + ((int64_t(window + local) << log_groups) + blockIdx.x) * d, d, from, scale, add);
        }
        // the others, and zeros for those that do not occur (after them it took 17% longer: 206 us in place of 176 for 1.07 GB)
        for (int local = warp; local < here; local += WARPS) {
            const int positions = counts[local];
            if (positions > AT_ONCE || (add && !positions)) continue;
            float acc[COLS][VEC] = {};
            if (positions) {
                int position = 0, held = 0;
                for (int w = 0; w < WARPS && held < positions; ++w)
                    for (int base = 0; base < length[w]; base += 32) held += take(w, base, local, position, held);
                add_rows<T, VEC, COLS>(acc, dy, d, from, position, positions);
            }
            store_row<O, VEC, COLS>(acc, dtable + ((int64_t(window + local) << log_groups) + blockIdx.x) * d, d, from, positions ? scale : 0.f, add);
        }
        workers_meet<THREADS>();
        if (own - window <= OWN) break;
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
constexpr int WIDE = 2, NARROW = 8;  // loads a lane for a gradient's part of a row: of 8 elements, or of one
// the way without groups (its grid has a part of a row for each second index)
bool few(const mimk_embedding_desc& d) { return d.n <= FEW && d.d <= int64_t(65535) * 32 * NARROW; }
Groups groups_in(Space& space, const mimk_embedding_desc& d) {
    Groups g{};
    if (few(d)) return g;
    g.count = static_cast<int*>(space.take(size_t(d.v) * 4)), g.start = static_cast<int*>(space.take(size_t(d.v) * 4));
    g.slot = static_cast<int*>(space.take(size_t(d.n) * 4)), g.order = static_cast<int*>(space.take(size_t(d.n) * 4));
    g.sorted = static_cast<int*>(space.take(size_t(d.n) * 4));
    // (a class of more than PIECE positions has less than twice as many pieces as it has whole ones)
    g.heavy = static_cast<int4*>(space.take((size_t(d.n) / LIGHT + size_t(d.n) / PIECE) * 16));
    g.part_pitch = up(d.d, 8), g.part = static_cast<float*>(space.take(size_t(d.n) / PIECE * 2 * size_t(g.part_pitch) * 4));
    g.light = static_cast<int*>(space.take(size_t(d.n) * 4));
    g.wholes = d.n / LIGHT, g.whole = static_cast<int*>(space.take(size_t(g.wholes) * 4));
    g.cursor = static_cast<int*>(space.take(CURSORS * 4));
    return g;
}

int check(const mimk_embedding_desc* d) {
    if (!d || d->n < 0 || d->d < 0 || d->v < 0) return MIMK_E_ARG;
    if ((d->dtype != MIMK_F32 && d->dtype != MIMK_BF16) || (d->out_dtype != MIMK_F32 && d->out_dtype != MIMK_BF16)) return MIMK_E_DTYPE;
    if (d->id_dtype != MIMK_I32 && d->id_dtype != MIMK_I64) return MIMK_E_DTYPE;
    if (d->n >= LIM - WINDOW || d->d >= LIM || d->v >= LIM) return MIMK_E_UNSUPPORTED;
    return MIMK_OK;
}
bool off(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % dtype_size(dtype) != 0; }
Ids ids_of(const mimk_embedding_desc& d) { return {d.ids, d.ignore_index, d.v, d.id_dtype == MIMK_I64, d.has_ignore != 0}; }
unsigned blocks_for(int64_t units, int64_t each, int64_t most) {
    const int64_t b = (units + each - 1) / each;
    return unsigned(b < 1 ? 1 : b < most ? b : most);
}

template <int VEC, int COLS>
int parts_of(int64_t d) {
    return int((d + 32 * VEC * COLS - 1) / (32 * VEC * COLS));
}
int log_up(int64_t v) {
    int log = 0;
    while ((int64_t(1) << log) < v) ++log;
    return log;
}
template <class T, class O, int VEC, int COLS>
int rows(const mimk_embedding_desc& d, const DeviceInfo& dev, cudaStream_t s) {
    constexpr int LOADS = VEC == 1 ? COLS : 2 * COLS;
    const int shift     = log_up(parts_of<VEC, LOADS>(d.d));
    return launch_after(rows_kernel<T, O, VEC, LOADS>, blocks_for(d.n << shift, WARPS, 1 << 20), THREADS, 0, s, static_cast<const T*>(d.table), ids_of(d), static_cast<O*>(d.out), d.n,
                        d.d, shift, d.scale, dev.status_dev);
}
template <class T, class O, int VEC, int COLS>
int grad(const mimk_embedding_desc& d, const Groups& g, const DeviceInfo& dev, cudaStream_t s) {
    const int parts = parts_of<VEC, COLS>(d.d);
    if (few(d)) {
        // Eight blocks to an SM, but no more groups than classes. 2048 positions here and 3000 the other way: 131072 x 4096 bf16 191 and 185 us, 50021 x 2048 54 and 62,
        // 10007 x 777 f32 28 and 62, 1000 x 4096 25 and 36, 131072 x 64 28 and 32.
        int log = 0;
        while ((int64_t(1) << (log + 1)) * parts <= int64_t(dev.sm_count) * 8 && (int64_t(1) << (log + 1)) <= d.v) ++log;
        return launch_after(few_kernel<T, O, VEC, COLS>, dim3(1u << log, unsigned(parts)), THREADS, 0, s, static_cast<const T*>(d.dy), ids_of(d), static_cast<O*>(d.dtable), int(d.n), d.d,
                            int(d.v), log, d.scale, d.add != 0, dev.status_dev);
    }
    MIMK_TRY(launch_after(clear_kernel, blocks_for(d.v, THREADS, int64_t(dev.sm_count) * 8), THREADS, 0, s, g, d.v));
    cudaLaunchAttribute together = {};
    together.id = cudaLaunchAttributeCooperative, together.val.cooperative = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(unsigned(dev.sm_count)), config.blockDim = dim3(BLOCK),  // (one to an SM)
    config.stream = s, config.attrs = &together, config.numAttrs = 1;
    return note_cuda_error(cudaLaunchKernelEx(&config, grad_kernel<T, O, VEC, COLS>, static_cast<const T*>(d.dy), ids_of(d), g, static_cast<O*>(d.dtable), d.n, d.d, d.v,
                                              log_up(parts), d.scale, d.add != 0, dev.status_dev));
}
// f<T, O, VEC, COLS>: by the element types, and whether rows are whole 16 bytes that start on such
#define MIMK_BY_TYPES(F, ALIGNED, ...)                                                                                                        \
    do {                                                                                                                                      \
        const bool f32_in = d->dtype == MIMK_F32, f32_out = d->out_dtype == MIMK_F32;                                                         \
        if (ALIGNED) {                                                                                                                        \
            if (f32_in) return f32_out ? F<float, float, 8, WIDE>(__VA_ARGS__) : F<float, __nv_bfloat16, 8, WIDE>(__VA_ARGS__);                \
            return f32_out ? F<__nv_bfloat16, float, 8, WIDE>(__VA_ARGS__) : F<__nv_bfloat16, __nv_bfloat16, 8, WIDE>(__VA_ARGS__);            \
        }                                                                                                                                     \
        if (f32_in) return f32_out ? F<float, float, 1, NARROW>(__VA_ARGS__) : F<float, __nv_bfloat16, 1, NARROW>(__VA_ARGS__);                \
        return f32_out ? F<__nv_bfloat16, float, 1, NARROW>(__VA_ARGS__) : F<__nv_bfloat16, __nv_bfloat16, 1, NARROW>(__VA_ARGS__);            \
    } while (0)

}  // namespace
}  // namespace mimk

using namespace mimk;

extern "C" int mimk_embedding(const mimk_embedding_desc* d, void* stream) {
    MIMK_TRY(check(d));
    int st                = MIMK_OK;
    const DeviceInfo* dev = device_info(&st);
    if (!dev) return st;
    if (!d->n || !d->d) return MIMK_OK;
    if ((!d->table && d->v) || !d->ids || !d->out) return MIMK_E_ARG;
    if (off(d->table, d->dtype) || off(d->out, d->out_dtype) || off(d->ids, d->id_dtype)) return MIMK_E_ALIGN;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    MIMK_BY_TYPES(rows, d->d % 8 == 0 && aligned16(d->table) && aligned16(d->out), *d, *dev, s);
}

extern "C" int mimk_embedding_grad_workspace(const mimk_embedding_desc* d, uint64_t* bytes) {
    MIMK_TRY(check(d));
    if (!bytes) return MIMK_E_ARG;
    Space space(nullptr);
    groups_in(space, *d);
    *bytes = space.used();
    return MIMK_OK;
}

extern "C" int mimk_embedding_grad(const mimk_embedding_desc* d, void* stream) {
    MIMK_TRY(check(d));
    int st                = MIMK_OK;
    const DeviceInfo* dev = device_info(&st);
    if (!dev) return st;
    if (!d->v || !d->d) return MIMK_OK;
    if (!d->dtable || (d->n && (!d->ids || !d->dy))) return MIMK_E_ARG;
    if (off(d->dy, d->dtype) || off(d->dtable, d->out_dtype) || off(d->ids, d->id_dtype)) return MIMK_E_ALIGN;
    Space space(d->workspace);
    const Groups g = groups_in(space, *d);
    if (space.used() > d->workspace_bytes || (space.used() && !d->workspace)) return MIMK_E_WORKSPACE;
    if (space.used() && !aligned16(d->workspace)) return MIMK_E_ALIGN;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    MIMK_BY_TYPES(grad, d->d % 8 == 0 && aligned16(d->dy) && aligned16(d->dtable), *d, g, *dev, s);
}
