// Token embedding and its gradient:  out[i] = scale table[ids[i]],   dtable[c] = scale sum over ids[i] = c of dy[i].
//
// The first is a copy of rows. For the second the positions are put in groups by class, without a sort: counted per class with integer atomics, a place
// for each class's group taken from a cursor, each position written to its group. Atomics leave a group's positions in any order, but their
// set is known, so each group is put in rising order before it is summed (32 positions by a warp, in registers; more of them by a block, as a map of
// bits), and results are the same call after call. A warp then owns 32 x VEC x COLS columns of a class: it adds up to 32 rows of dy, or writes zeros;
// classes of more rows are taken by whole blocks, a run of the rows for each warp, joined in shared memory.
// What bounds it: the bytes, most of all the table's gradient.
#include "elements.cuh"
#include "train_common.cuh"

namespace mimk {

namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int LIGHT = 32;            // positions of a class that one warp adds up
constexpr int WINDOW = 1 << 17;      // positions in one map of bits
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

// COLS loads of VEC elements, 32 lanes side by side, are a part of a row: one warp's work.
template <class T, class O, int VEC, int COLS>
__global__ void __launch_bounds__(THREADS) rows_kernel(const T* table, Ids ids, O* out, int64_t n, int64_t d, int parts, float scale, int* status) {
    after_previous();
    const int lane = threadIdx.x & 31;
    const int64_t units = n * parts;
    for (int64_t u = int64_t(blockIdx.x) * WARPS + (threadIdx.x >> 5); u < units; u += int64_t(gridDim.x) * WARPS) {
        const int64_t i = parts == 1 ? u : u / parts;
        const int64_t from = (u - i * parts) * (32 * VEC * COLS) + lane * VEC;
        const int c = class_at(ids, i);
        if (c == BAD && lane == 0) *status = MIMK_E_SHAPE;
        Run<T, VEC> run[COLS];
#pragma unroll
        for (int k = 0; k < COLS; ++k) {
            const int64_t at = from + k * 32 * VEC;
            run[k].clear();
            if (c >= 0 && at < d) run[k].load(table + int64_t(c) * d + at);
        }
#pragma unroll
        for (int k = 0; k < COLS; ++k) {
            const int64_t at = from + k * 32 * VEC;
            if (at >= d) break;
            float v[VEC];
            run[k].get(v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = c == BAD ? NAN : c == NO_TOKEN ? 0.f : v[j] * scale;
            put(out + i * d + at, v);
        }
    }
}

// ---- groups ------------------------------------------------------------------------------------------------------------------------
struct Groups {
    int* count;   // [v] positions of a class
    int* start;   // [v] where its group begins
    int* slot;    // [n] place in the group, in any order
    int* order;   // [n] positions by group
    int* sorted;  // [n] the same, groups of more than LIGHT positions in rising order
    int* heavy;   // [n / LIGHT] classes of such groups
    int* cursor;  // places taken; heavy classes
};

__global__ void __launch_bounds__(THREADS) clear_kernel(Groups g, int64_t v) {
    after_previous();
    if (blockIdx.x == 0 && threadIdx.x < 2) g.cursor[threadIdx.x] = 0;
    for (int64_t i = int64_t(blockIdx.x) * THREADS + threadIdx.x; i < v; i += int64_t(gridDim.x) * THREADS) g.count[i] = 0;
}

__global__ void __launch_bounds__(THREADS) count_kernel(Ids ids, Groups g, int64_t n, int* status) {
    after_previous();
    for (int64_t base = int64_t(blockIdx.x) * THREADS; base < n; base += int64_t(gridDim.x) * THREADS) {
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
    __shared__ int part[WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int sum = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int w = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += w;
    }
    __syncthreads();  // (of an earlier call's reads)
    if (lane == 31) part[warp] = sum;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        before += w < warp ? part[w] : 0;
        all += part[w];
    }
    *total = all;
    return before + sum - v;
}

__global__ void __launch_bounds__(THREADS) start_kernel(Groups g, int64_t v) {
    __shared__ int first[2];
    after_previous();
    for (int64_t base = int64_t(blockIdx.x) * THREADS; base < v; base += int64_t(gridDim.x) * THREADS) {
        const int64_t c = base + threadIdx.x;
        const int count = c < v ? g.count[c] : 0;
        int all, heavies;
        const int before = block_before(count, &all), nth = block_before(count > LIGHT, &heavies);
        if (!all) continue;
        if (threadIdx.x == 0) first[0] = atomicAdd(g.cursor, all), first[1] = heavies ? atomicAdd(g.cursor + 1, heavies) : 0;
        __syncthreads();
        if (count) g.start[c] = first[0] + before;
        if (count > LIGHT) g.heavy[first[1] + nth] = int(c);
        __syncthreads();
    }
}

__global__ void __launch_bounds__(THREADS) place_kernel(Ids ids, Groups g, int64_t n) {
    after_previous();
    for (int64_t i = int64_t(blockIdx.x) * THREADS + threadIdx.x; i < n; i += int64_t(gridDim.x) * THREADS) {
        const int slot = g.slot[i];
        if (slot >= 0) g.order[g.start[class_at(ids, i)] + slot] = int(i);
    }
}

// A block for a heavy class: its positions as bits of a map, read off in order.
__global__ void __launch_bounds__(THREADS) sort_kernel(Groups g, int64_t n) {
    __shared__ uint32_t bits[WINDOW / 32];
    after_previous();
    const int heavies = g.cursor[1];
    for (int h = blockIdx.x; h < heavies; h += gridDim.x) {
        const int c = g.heavy[h], count = g.count[c], start = g.start[c];
        int done = 0;
        for (int64_t window = 0; window < n && done < count; window += WINDOW) {
            const int words = int(n - window < WINDOW ? (n - window + 31) / 32 : WINDOW / 32);
            const int each  = (words + THREADS - 1) / THREADS;
            for (int w = threadIdx.x; w < words; w += THREADS) bits[w] = 0;
            __syncthreads();
            for (int k = threadIdx.x; k < count; k += THREADS) {
                const int64_t at = g.order[start + k] - window;
                if (at >= 0 && at < WINDOW) atomicOr(bits + (at >> 5), 1u << (at & 31));
            }
            __syncthreads();
            const int lo = min(words, int(threadIdx.x) * each), hi = min(words, lo + each);
            int mine = 0, all;
            for (int w = lo; w < hi; ++w) mine += __popc(bits[w]);
            int to = start + done + block_before(mine, &all);
            for (int w = lo; w < hi; ++w)
                for (uint32_t b = bits[w]; b; b &= b - 1) g.sorted[to++] = int(window) + w * 32 + __ffs(b) - 1;
            done += all;
            __syncthreads();
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
template <class O, int VEC, int COLS>
__device__ __forceinline__ void store_row(const float (&acc)[COLS][VEC], O* row, int64_t d, int64_t from, float scale, bool add) {
#pragma unroll
    for (int q = 0; q < COLS; ++q) {
        const int64_t at = from + q * 32 * VEC;
        if (at >= d) break;
        float v[VEC], old[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) old[j] = 0.f;
        if (add) {
            Run<O, VEC> r;
            r.load(row + at), r.get(old);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = add ? fmaf(acc[q][j], scale, old[j]) : acc[q][j] * scale;
        put(row + at, v);
    }
}

template <class T, class O, int VEC, int COLS>
__global__ void __launch_bounds__(THREADS) sum_kernel(const T* dy, Groups g, O* dtable, int64_t d, int64_t v, int parts, float scale, bool add) {
    constexpr int PART = 32 * VEC * COLS;
    __shared__ float joined[WARPS][PART];
    after_previous();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t heavy_units = int64_t(g.cursor[1]) * parts;
    for (int64_t u = blockIdx.x; u < heavy_units; u += gridDim.x) {
        const int64_t h    = u / parts;
        const int64_t from = (u - h * parts) * PART + lane * VEC;
        const int c = g.heavy[h], count = g.count[c], start = g.start[c];
        const int each = (count + WARPS - 1) / WARPS, lo = min(count, warp * each), hi = min(count, lo + each);
        float acc[COLS][VEC] = {};
        for (int k = lo; k < hi; k += 32) add_rows<T, VEC, COLS>(acc, dy, d, from, k + lane < hi ? g.sorted[start + k + lane] : 0, min(32, hi - k));
#pragma unroll
        for (int q = 0; q < COLS; ++q)
#pragma unroll
            for (int j = 0; j < VEC; ++j) joined[warp][(q * VEC + j) * 32 + lane] = acc[q][j];
        __syncthreads();
        if (warp == 0) {
#pragma unroll
            for (int q = 0; q < COLS; ++q)
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    for (int w = 1; w < WARPS; ++w) acc[q][j] += joined[w][(q * VEC + j) * 32 + lane];
            store_row<O, VEC, COLS>(acc, dtable + int64_t(c) * d, d, from, scale, add);
        }
        __syncthreads();
    }
    // the other classes: units warp, warp + warps, ...; what 32 of them need to know comes in one load each
    const int64_t units = v * parts, warps = int64_t(gridDim.x) * WARPS;
    for (int64_t first = int64_t(blockIdx.x) * WARPS + warp; first < units; first += 32 * warps) {
        const int64_t mine = first + lane * warps;
        const int count    = mine < units ? g.count[mine / parts] : -1;
        const int start    = count > 0 && count <= LIGHT ? g.start[mine / parts] : 0;
        for (unsigned left = __ballot_sync(0xffffffffu, count >= 0 && count <= LIGHT && !(add && count == 0)); left; left &= left - 1) {
            const int k        = __ffs(left) - 1;
            const int64_t u    = first + k * warps, c = u / parts;
            const int64_t from = (u - c * parts) * PART + lane * VEC;
            const int positions = __shfl_sync(0xffffffffu, count, k), begin = __shfl_sync(0xffffffffu, start, k);
            float acc[COLS][VEC] = {};
            if (positions) add_rows<T, VEC, COLS>(acc, dy, d, from, sorted_lanes(lane < positions ? g.order[begin + lane] : INT_MAX), positions);
            store_row<O, VEC, COLS>(acc, dtable + c * d, d, from, positions ? scale : 0.f, add);
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
Groups groups_in(Space& space, const mimk_embedding_desc& d) {
    Groups g;
    g.count = static_cast<int*>(space.take(size_t(d.v) * 4)), g.start = static_cast<int*>(space.take(size_t(d.v) * 4));
    g.slot = static_cast<int*>(space.take(size_t(d.n) * 4)), g.order = static_cast<int*>(space.take(size_t(d.n) * 4));
    g.sorted = static_cast<int*>(space.take(size_t(d.n) * 4)), g.heavy = static_cast<int*>(space.take(size_t(d.n) / LIGHT * 4));
    g.cursor = static_cast<int*>(space.take(8));
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

constexpr int WIDE = 2, NARROW = 8;  // loads a lane: of 8 elements, or of one

template <class T, class O, int VEC, int COLS>
int rows(const mimk_embedding_desc& d, const DeviceInfo& dev, cudaStream_t s) {
    const int parts = int((d.d + 32 * VEC * COLS - 1) / (32 * VEC * COLS));
    return launch_after(rows_kernel<T, O, VEC, COLS>, blocks_for(d.n * parts, WARPS, 1 << 20), THREADS, 0, s, static_cast<const T*>(d.table), ids_of(d),
                        static_cast<O*>(d.out), d.n, d.d, parts, d.scale, dev.status_dev);
}
template <class T, class O, int VEC, int COLS>
int sums(const mimk_embedding_desc& d, const Groups& g, const DeviceInfo& dev, cudaStream_t s) {
    const int parts = int((d.d + 32 * VEC * COLS - 1) / (32 * VEC * COLS));
    return launch_after(sum_kernel<T, O, VEC, COLS>, blocks_for(d.v * parts, WARPS, int64_t(dev.sm_count) * 4), THREADS, 0, s, static_cast<const T*>(d.dy), g,
                        static_cast<O*>(d.dtable), d.d, d.v, parts, d.scale, d.add != 0);
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
    if (!d->workspace || space.used() > d->workspace_bytes) return MIMK_E_WORKSPACE;
    if (!aligned16(d->workspace)) return MIMK_E_ALIGN;
    cudaStream_t s     = static_cast<cudaStream_t>(stream);
    const int64_t most = int64_t(dev->sm_count) * 8;
    const Ids ids      = ids_of(*d);
    MIMK_TRY(launch_after(clear_kernel, blocks_for(d->v, THREADS, most), THREADS, 0, s, g, d->v));
    if (d->n) {
        MIMK_TRY(launch_after(count_kernel, blocks_for(d->n, THREADS, most), THREADS, 0, s, ids, g, d->n, dev->status_dev));
        MIMK_TRY(launch_after(start_kernel, blocks_for(d->v, THREADS, most), THREADS, 0, s, g, d->v));
        MIMK_TRY(launch_after(place_kernel, blocks_for(d->n, THREADS, most), THREADS, 0, s, ids, g, d->n));
        if (d->n > LIGHT) MIMK_TRY(launch_after(sort_kernel, blocks_for(d->n, LIGHT + 1, most / 2), THREADS, 0, s, g, d->n));
    }
    MIMK_BY_TYPES(sums, d->d % 8 == 0 && aligned16(d->dy) && aligned16(d->dtable), *d, g, *dev, s);
}
