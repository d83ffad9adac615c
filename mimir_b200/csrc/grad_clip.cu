// The 2-norm of a list of gradients, and their clipping:  norm = sqrt(sum over all tensors of g^2),  out = g min(1, limit / (norm + eps)).
//
// Two launches over a table of the tensors (a kernel's parameter: up to 1024 of them at once). The tensors are cut into chunks of 32 KiB that start
// on 16-byte boundaries; CTAs take the chunks in turn. The first launch leaves one sum per CTA; each CTA of the second adds those up itself, always in
// the same order, and scales its chunks, the last ones first: what of the gradients the L2 cache still holds comes from there.
// What bounds it: the bytes, twice read and once written: 345 MB of bf16 into other tensors 163 to 170 us, 6.2 TB/s of 1.03 GB; the norm alone 54. In
// place, tensors whose norm is within the limit are left alone. Results at another offset from 16 bytes than their tensor go value by value: 1.10 ms
// for the same (f32: 1.22 where 0.32).
#include "common.cuh"

namespace mimk {

namespace {

constexpr int CHUNK = 32768, THREADS = 256, LOADS = CHUNK / (THREADS * 16);
constexpr int MOST_CTAS = 8;  // per SM

template <int N>
struct Table {
    const void* in[N];
    void* out[N];
    int64_t bytes[N];
    int first[N + 1];             // first chunk of each tensor
    uint32_t f32[(N + 31) / 32];  // a bit per tensor: f32, or bf16
    int count;
};

struct Chunk {
    const uint8_t* in;
    uint8_t* out;
    int from, to;   // bytes from `in` that belong to the tensor
    bool f32;
};
// The tensor that a chunk lies in, by halving; the chunk starts at a multiple of 16 bytes, at or before the tensor's first byte.
template <int N>
__device__ __forceinline__ Chunk chunk_at(const Table<N>& t, int at) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= at) lo = mid;
        else hi = mid - 1;
    }
    const uintptr_t p   = reinterpret_cast<uintptr_t>(t.in[lo]);
    const int lead      = int(p & 15);
    const int64_t start = int64_t(at - t.first[lo]) * CHUNK - lead;  // of the chunk, in bytes from the tensor's first
    Chunk c;
    c.in   = static_cast<const uint8_t*>(t.in[lo]) + start;
    c.out  = static_cast<uint8_t*>(t.out[lo]) + start;
    c.from = start < 0 ? lead : 0;
    c.to   = int(t.bytes[lo] - start < CHUNK ? t.bytes[lo] - start : CHUNK);
    c.f32  = (t.f32[lo >> 5] >> (lo & 31)) & 1;
    return c;
}

__device__ __forceinline__ float low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// The squares of up to 16 values, as f64: summed in f32, and again in f64 where that overflows, or where the squares are so small that bits of
// them may be lost.
template <bool F32, int W>
__device__ __forceinline__ double squares(const uint32_t (&w)[W]) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        if (F32) s = fmaf(__uint_as_float(w[i]), __uint_as_float(w[i]), s);
        else s = fmaf(high(w[i]), high(w[i]), fmaf(low(w[i]), low(w[i]), s));
    }
    if (s > 1e-25f && s < INFINITY) return double(s);
    double d = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        if (F32) d += double(__uint_as_float(w[i])) * double(__uint_as_float(w[i]));
        else d += double(low(w[i])) * double(low(w[i])) + double(high(w[i])) * double(high(w[i]));
    }
    return d;
}

// Single values at a chunk's ends.
template <bool F32>
__device__ __forceinline__ uint32_t word_at(const uint8_t* p, int at) {
    return F32 ? *reinterpret_cast<const uint32_t*>(p + at) : uint32_t(*reinterpret_cast<const uint16_t*>(p + at)) << 16;
}

template <bool F32>
__device__ __forceinline__ double chunk_squares(const Chunk& c) {
    constexpr int SIZE = F32 ? 4 : 2;
    const int head = min((c.from + 15) & ~15, c.to), tail = max(head, c.to & ~15);
    double sum     = 0;
    uint4 v[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int at = head + (i * THREADS + int(threadIdx.x)) * 16;
        v[i]         = at < tail ? *reinterpret_cast<const uint4*>(c.in + at) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < LOADS; i += F32 ? 4 : 2) {
        if (head + (i * THREADS + int(threadIdx.x)) * 16 >= tail) break;
        if (F32) {
            const uint32_t w[16] = {v[i].x,     v[i].y,     v[i].z,     v[i].w,     v[i + 1].x, v[i + 1].y, v[i + 1].z, v[i + 1].w,
                                    v[i + 2].x, v[i + 2].y, v[i + 2].z, v[i + 2].w, v[i + 3].x, v[i + 3].y, v[i + 3].z, v[i + 3].w};
            sum += squares<true>(w);
        } else {
            const uint32_t w[8] = {v[i].x, v[i].y, v[i].z, v[i].w, v[i + 1].x, v[i + 1].y, v[i + 1].z, v[i + 1].w};
            sum += squares<false>(w);
        }
    }
    const int before = (head - c.from) / SIZE, behind = (c.to - tail) / SIZE;
    if (int(threadIdx.x) < before + behind) {
        const int at = int(threadIdx.x) < before ? c.from + int(threadIdx.x) * SIZE : tail + (int(threadIdx.x) - before) * SIZE;
        const double d = double(__uint_as_float(word_at<F32>(c.in, at)));
        sum += d * d;
    }
    return sum;
}

__device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[THREADS / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) v += part[w];
    return v;
}

template <int N>
__global__ void __launch_bounds__(THREADS) squares_kernel(const __grid_constant__ Table<N> t, double* __restrict__ sums) {
    after_previous();
    double sum      = 0;
    const int total = t.first[t.count];
    for (int at = blockIdx.x; at < total; at += gridDim.x) {
        const Chunk c = chunk_at(t, at);
        sum += c.f32 ? chunk_squares<true>(c) : chunk_squares<false>(c);
    }
    sum = block_sum(sum);
    if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

// every CTA adds up all sums, a thread every THREADS-th of them
__device__ __forceinline__ double total_of(const double* sums, int count) {
    double s = 0;
    for (int i = threadIdx.x; i < count; i += THREADS) s += sums[i];
    return sqrt(block_sum(s));
}
__global__ void __launch_bounds__(THREADS) norm_kernel(const double* sums, int count, float* norm) {
    after_previous();
    const double n = total_of(sums, count);
    if (threadIdx.x == 0) *norm = float(n);
}

template <bool F32>
__device__ __forceinline__ uint32_t scaled(uint32_t w, float c) {
    if (F32) return __float_as_uint(__uint_as_float(w) * c);
    return pack_bf16x2(low(w) * c, high(w) * c);
}
template <bool F32>
__device__ __forceinline__ void scale_one(const Chunk& c, int at, float by) {
    const float v = __uint_as_float(word_at<F32>(c.in, at)) * by;
    if (F32) *reinterpret_cast<float*>(c.out + at) = v;
    else *reinterpret_cast<__nv_bfloat16*>(c.out + at) = __float2bfloat16(v);
}
template <bool F32>
__device__ __forceinline__ void scale_chunk(const Chunk& c, float by) {
    constexpr int SIZE = F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(c.out) & 15) {  // the result lies otherwise than the tensor
        for (int at = c.from + int(threadIdx.x) * SIZE; at < c.to; at += THREADS * SIZE) scale_one<F32>(c, at, by);
        return;
    }
    const int head = min((c.from + 15) & ~15, c.to), tail = max(head, c.to & ~15);
    uint4 v[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int at = head + (i * THREADS + int(threadIdx.x)) * 16;
        if (at < tail) v[i] = *reinterpret_cast<const uint4*>(c.in + at);
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int at = head + (i * THREADS + int(threadIdx.x)) * 16;
        if (at < tail)
            __stcs(reinterpret_cast<uint4*>(c.out + at),
                   make_uint4(scaled<F32>(v[i].x, by), scaled<F32>(v[i].y, by), scaled<F32>(v[i].z, by), scaled<F32>(v[i].w, by)));
    }
    const int before = (head - c.from) / SIZE, behind = (c.to - tail) / SIZE;
    if (int(threadIdx.x) < before + behind)
        scale_one<F32>(c, int(threadIdx.x) < before ? c.from + int(threadIdx.x) * SIZE : tail + (int(threadIdx.x) - before) * SIZE, by);
}

template <int N>
__global__ void __launch_bounds__(THREADS) scale_kernel(const __grid_constant__ Table<N> t, const double* sums, int n_sums, double limit, double eps,
                                                       float* norm, bool in_place) {
    after_previous();
    const double n = total_of(sums, n_sums);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = float(n);
    const double c = limit / (n + eps);
    const float by = c >= 1 ? 1.f : float(c);  // (NaN stays NaN)
    if (in_place && by == 1.f) return;
    for (int at = t.first[t.count] - 1 - int(blockIdx.x); at >= 0; at -= gridDim.x) {
        const Chunk chunk = chunk_at(t, at);
        if (chunk.f32) scale_chunk<true>(chunk, by);
        else scale_chunk<false>(chunk, by);
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
constexpr int SMALL = 64, LARGE = 1024;

struct List {
    const void* const* in;
    void* const* out;
    const int64_t* lengths;
    const int32_t* dtypes;
    int64_t count;
};
size_t size_of(int dtype) { return dtype == MIMK_BF16 ? 2 : 4; }

int check(const List& l, bool pointers) {
    if (l.count < 0 || (l.count > 0 && (!l.lengths || !l.dtypes || (pointers && !l.in)))) return MIMK_E_ARG;
    for (int64_t i = 0; i < l.count; ++i) {
        if (l.dtypes[i] != MIMK_F32 && l.dtypes[i] != MIMK_BF16) return MIMK_E_DTYPE;
        if (l.lengths[i] < 0) return MIMK_E_ARG;
        if (l.lengths[i] >= int64_t(1) << 44) return MIMK_E_UNSUPPORTED;
        if (!pointers || !l.lengths[i]) continue;
        if (!l.in[i] || (l.out && !l.out[i])) return MIMK_E_ARG;
        if (reinterpret_cast<uintptr_t>(l.in[i]) % size_of(l.dtypes[i]) || (l.out && reinterpret_cast<uintptr_t>(l.out[i]) % size_of(l.dtypes[i]))) return MIMK_E_ALIGN;
    }
    return MIMK_OK;
}

// f(table, first sum, CTAs) for each run of up to N tensors that are not empty; how many sums there are in all
template <int N, class F>
int each_table(const List& l, int sm_count, F&& f) {
    static thread_local Table<N> t;  // (24 KiB)
    int sums  = 0;
    int64_t i = 0;
    while (i < l.count) {
        t.count       = 0;
        int64_t total = 0;
        for (uint32_t& w : t.f32) w = 0;
        for (; i < l.count && t.count < N; ++i) {
            if (!l.lengths[i]) continue;
            const int64_t bytes  = l.lengths[i] * int64_t(size_of(l.dtypes[i]));
            const int64_t chunks = (int64_t(reinterpret_cast<uintptr_t>(l.in[i]) & 15) + bytes + CHUNK - 1) / CHUNK;
            if (total + chunks > (1 << 30)) {
                if (!t.count) return MIMK_E_UNSUPPORTED;
                break;
            }
            t.in[t.count] = l.in[i], t.out[t.count] = l.out ? l.out[i] : nullptr, t.bytes[t.count] = bytes, t.first[t.count] = int(total);
            if (l.dtypes[i] == MIMK_F32) t.f32[t.count >> 5] |= 1u << (t.count & 31);
            total += chunks, ++t.count;
        }
        if (!t.count) break;
        t.first[t.count] = int(total);
        const int64_t most = int64_t(sm_count) * MOST_CTAS;
        const int ctas     = int(total < most ? total : most);
        MIMK_TRY(f(t, sums, ctas));
        sums += ctas;
    }
    return MIMK_OK;
}

int64_t tables_of(int64_t count) { return count <= SMALL ? 1 : (count + LARGE - 1) / LARGE; }
// (a table ends early only where its tensors have 2^30 chunks: a run of 32 TiB)
uint64_t workspace_of(int64_t count, int sm_count) { return uint64_t(tables_of(count) + 1) * uint64_t(sm_count) * MOST_CTAS * 8; }

template <int N>
int run(const List& l, const DeviceInfo& dev, bool clip, float limit, float eps, float* norm, double* sums, cudaStream_t s) {
    int all = 0;
    MIMK_TRY((each_table<N>(l, dev.sm_count, [&](const Table<N>& t, int first, int ctas) {
        all = first + ctas;
        return launch_after(squares_kernel<N>, unsigned(ctas), THREADS, 0, s, t, sums + first);
    })));
    if (!clip || !all) {
        return launch_after(norm_kernel, 1, THREADS, 0, s, static_cast<const double*>(sums), all, norm);
    }
    bool in_place = true;
    for (int64_t i = 0; i < l.count; ++i) in_place = in_place && (!l.lengths[i] || l.in[i] == l.out[i]);
    return each_table<N>(l, dev.sm_count, [&](const Table<N>& t, int first, int ctas) {
        return launch_after(scale_kernel<N>, unsigned(ctas), THREADS, 0, s, t, static_cast<const double*>(sums), all, double(limit), double(eps), first ? nullptr : norm,
                            bool(in_place));
    });
}

int entry(const List& l, bool clip, float limit, float eps, float* norm, void* workspace, uint64_t bytes, void* stream) {
    MIMK_TRY(check(l, true));
    if (clip && l.count > 0 && !l.out) return MIMK_E_ARG;
    if (clip && (!(limit >= 0) || !(eps >= 0))) return MIMK_E_ARG;
    if (!norm) return MIMK_E_ARG;
    int st                = MIMK_OK;
    const DeviceInfo* dev = device_info(&st);
    if (!dev) return st;
    if (!workspace || bytes < workspace_of(l.count, dev->sm_count)) return MIMK_E_WORKSPACE;
    if (!aligned16(workspace)) return MIMK_E_ALIGN;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    double* sums   = static_cast<double*>(workspace);
    // (a small table is 2 KiB of parameters for each launch, a large one 28)
    return l.count <= SMALL ? run<SMALL>(l, *dev, clip, limit, eps, norm, sums, s) : run<LARGE>(l, *dev, clip, limit, eps, norm, sums, s);
}

}  // namespace
}  // namespace mimk

using namespace mimk;

extern "C" int mimk_clip_grads_workspace(int64_t count, uint64_t* bytes) {
    if (count < 0 || !bytes) return MIMK_E_ARG;
    int st                = MIMK_OK;
    const DeviceInfo* dev = device_info(&st);
    if (!dev) return st;
    *bytes = workspace_of(count, dev->sm_count);
    return MIMK_OK;
}
extern "C" int mimk_grad_norm(const void* const* tensors, const int64_t* lengths, const int32_t* dtypes, int64_t count, float* norm, void* workspace,
                              uint64_t workspace_bytes, void* stream) {
    return entry({tensors, nullptr, lengths, dtypes, count}, false, 0.f, 0.f, norm, workspace, workspace_bytes, stream);
}
extern "C" int mimk_clip_grads(const void* const* tensors, void* const* out, const int64_t* lengths, const int32_t* dtypes, int64_t count, float limit, float eps,
                               float* norm, void* workspace, uint64_t workspace_bytes, void* stream) {
    return entry({tensors, out, lengths, dtypes, count}, true, limit, eps, norm, workspace, workspace_bytes, stream);
}
