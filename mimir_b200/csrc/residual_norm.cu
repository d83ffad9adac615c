// From one block of a model to the next, and its gradients:
//   u = e h post_gamma,  r_out = a r + b gate u,  x = s r_out gamma         e = 1 / sqrt(mean h^2 + eps),  s = 1 / sqrt(mean r_out^2 + eps)
//   t = dx gamma,  D = dr_out + s t - s^3 r_out mean(t r_out):  dr = a D,  dgamma = sum dx s r_out,  dgate = sum b u D
//   q = b gate post_gamma:  dpost_gamma = sum b gate e h D,  dh = e q D - e^3 h mean(q h D)
// A row belongs to a team of threads, a warp or a block, and stays in their registers, or is read twice (long rows backward). The backward pass has one join of sums for a row: with hats for
// e h and s r_out, and D = (dr_out + s t) - k r_out^,  k = s mean(t r_out^),  the second mean is mean(q h^ (dr_out + s t)) - k mean(q h^ r_out^). r_out is
// computed over again from r and h, the same bytes as reading it, so that a stream kept in bf16 is not rounded on the way into the gradients.
// Gradients over rows are summed by each team over its rows and over the teams by a second launch.
// What bounds it: the bytes, 8 of each value forward and 12 backward (bf16). 8192 x 4096 bf16, both norms and a gate: forward 55 us, 4.9 TB/s; backward 84 and the join of
// sums 7, 4.8 TB/s. One block's registers fill an SM, so that two teams of 256 threads forward, or one of 512 backward, wait for their sums with little beside them to do: 3300 cycles a row
// and team forward, 600 of them with an instruction to issue. Without a norm of h and a gate: 51 and 89 us. Rows held in registers, without a ring: 254 us for both passes.
#include "attn_common.cuh"
#include "elements.cuh"
#include "train_common.cuh"

namespace mimk {

namespace {

constexpr int64_t MOST_COLUMNS = 32768, LIM = (int64_t(1) << 31) - (1 << 17);  // (rows in 32 bits, with a team's step behind the last)

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
    // sums over rows: one row of d for each team, or (gate) for each unit of rows; a unit that is a whole group of the gate's writes dgate
    float *part_gamma, *part_post, *part_gate, *part_z;
    int shared;  // (backward_kernel) sums for each column are kept in shared memory
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

// VEC elements side by side, CH times, blockDim.x threads apart: what a thread holds of a row. (Two blocks of 512 threads to an SM: 8192 x 4096 off 16 bytes 231 us, one 352.)
template <class RT, class HT, int VEC, int CH, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT == 512 ? 2 : 1) forward_kernel(const __grid_constant__ Args<RT, HT> g) {
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
            e = rsqrtf(fmaf(sum[0], per, g.eps));
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
            s = rsqrtf(fmaf(sum[0], per, g.eps));
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

// A block for each row, which is read twice, the second time from the caches: what is kept from row to row, sums for each column, takes shared memory or, of longer rows, the block's
// rows of partial sums themselves, and no thread touches another's columns. (4096 x 16384 bf16: 285 us, 2.8 TB/s; with a row and the
// sums in registers, 32 columns a thread, which spilled, 957.)
constexpr int THREADS = 512;  // of a block: one team of all of them, or several
template <class RT, class HT, int VEC>
__global__ void __launch_bounds__(THREADS, 1) backward_kernel(const __grid_constant__ Args<RT, HT> g) {
    extern __shared__ __align__(16) float room[];
    after_previous();
    const int d = int(g.d), array = (d + 3) & ~3, t = threadIdx.x * VEC, step = blockDim.x * VEC;
    const float per       = 1.f / float(d);
    const bool several    = g.groups > 1;
    const int64_t own     = int64_t(blockIdx.x) * d;
    float* const dgamma   = g.shared ? room : g.part_gamma + own;
    float* const z        = g.shared ? room + array : (several ? g.part_z : g.part_post) + own;  // sum D h^: of the unit's rows, or of all
    float* const dpost    = g.shared ? room + 2 * array : g.part_post + own;
    const bool with_gamma = g.part_gamma != nullptr, with_z = g.post_gamma.p || g.gate.p, with_post = several && g.part_post != nullptr;
    const auto columns    = [&](auto&& f) {
        for (int at = t; at < d; at += step) f(at);
    };
    const auto add = [](float* to, const float (&v)[VEC]) {
        Run<float, VEC> run;
        float old[VEC];
        run.load(to), run.get(old);
#pragma unroll
        for (int j = 0; j < VEC; ++j) old[j] += v[j];
        put(to, old);
    };
    const float nothing[VEC] = {};
    columns([&](int at) {
        if (with_gamma) put(dgamma + at, nothing);
        if (with_z) put(z + at, nothing);
        if (with_post) put(dpost + at, nothing);
    });
    for (int64_t unit = blockIdx.x; unit < g.groups * g.pieces; unit += gridDim.x) {
        const int64_t group = unit / g.pieces, piece = unit - group * g.pieces, end = min(g.n, (group + 1) * g.gate_rows);
        for (int64_t row = group * g.gate_rows + piece; row < end; row += g.pieces) {
            const float e = g.post_gamma.p ? g.kept[row] : 1.f, s = g.gamma.p ? g.kept[g.n + row] : 1.f;
            // h^, r_out^, dr_out + s t, q, t and dx of a thread's columns
            float hat[VEC], rhat[VEC], before[VEC], q[VEC], w[VEC], dx[VEC];
            const auto read = [&](int at) {
                const int64_t p = row * g.d + at;
                Run<RT, VEC> rr, drr;
                Run<HT, VEC> hr, dxr;
                hr.clear(), drr.clear(), dxr.clear(), rr.load(g.r + p);
                if (g.h) hr.load(g.h + p);
                if (g.dr_out) drr.load(g.dr_out + p);
                if (g.dx) dxr.load(g.dx + p);
                float gate[VEC];
                factors_at(g.gamma, at, w), factors_at(g.post_gamma, at, q), factors_at(g.gate, group * g.d + at, gate);
                rr.get(rhat), hr.get(hat), drr.get(before), dxr.get(dx);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    q[j] *= g.b * gate[j], hat[j] *= e, w[j] *= dx[j];
                    rhat[j]   = g.h ? s * fmaf(g.a, rhat[j], q[j] * hat[j]) : s * rhat[j];
                    before[j] = fmaf(s, w[j], before[j]);
                }
            };
            float sum[3] = {};
            columns([&](int at) {
                read(at);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float qh = q[j] * hat[j];
                    sum[0] = fmaf(w[j], rhat[j], sum[0]), sum[1] = fmaf(qh, before[j], sum[1]), sum[2] = fmaf(qh, rhat[j], sum[2]);
                    dx[j] *= rhat[j];
                }
                if (with_gamma) add(dgamma + at, dx);
            });
            team_sum(sum);
            const float k = g.gamma.p ? s * sum[0] * per : 0.f, m = g.post_gamma.p ? (sum[1] - k * sum[2]) * per : 0.f;
            columns([&](int at) {
                read(at);
                float out[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float D = fmaf(-k, rhat[j], before[j]);
                    out[j] = g.a * D;
                    q[j]   = e * fmaf(q[j], D, -hat[j] * m);
                    hat[j] *= D;
                }
                put(g.dr + row * g.d + at, out);
                if (g.dh) put(g.dh + row * g.d + at, q);
                if (with_z) add(z + at, hat);
            });
        }
        if (several && with_z) {
            columns([&](int at) {
                Run<float, VEC> run;
                float sums[VEC], f[VEC], gate[VEC];
                run.load(z + at), run.get(sums), put(z + at, nothing);
                factors_at(g.post_gamma, at, f), factors_at(g.gate, group * g.d + at, gate);
#pragma unroll
                for (int j = 0; j < VEC; ++j) gate[j] *= g.b * sums[j], f[j] *= g.b * sums[j];
                if (with_post) add(dpost + at, gate);
                if (g.pieces > 1) put(g.part_gate + unit * g.d + at, f);
                else if (g.gate.bf16) put(static_cast<__nv_bfloat16*>(g.dgate) + group * g.d + at, f);
                else put(static_cast<float*>(g.dgate) + group * g.d + at, f);
            });
        }
    }
    if (!g.shared) return;
    columns([&](int at) {
        Run<float, VEC> run;
        float v[VEC];
        if (with_gamma) run.load(dgamma + at), run.get(v), put(g.part_gamma + own + at, v);
        if (g.part_post) run.load((several ? dpost : z) + at), run.get(v), put(g.part_post + own + at, v);
    });
}

// ---- the same with rows on their way in shared memory --------------------------------------------------------------------------------
// What a thread needs of the next rows is asked for up to six rows ahead: at the bytes that an SM gets, some 50 KiB have to be on their way for each, and 200 can be.
// Each thread copies the columns that are its own, into places of its own (cp.async), so that what is on its way takes no registers and no barrier.
// Columns are taken in chunks of eight that start on 16-byte boundaries: of a row that begins `lead` elements past one, the first chunk has the end of the row
// before it and the last one the beginning of the next, which are left out when values are read. With 8 / gcd(d, 8) classes of rows, a row's number modulo that count
// decides its lead: a team's rows are all of one class, so that its columns are the same in every row.
template <class T>
constexpr int PLANES = sizeof(T) * 8 / 16;  // 16-byte pieces of a chunk

__device__ __forceinline__ void copy_async(uint32_t to, const void* from, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// at most N groups of copies of this thread still on their way
template <int N>
__device__ __forceinline__ void copies_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 take16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void leave16(uint32_t at, float a, float b, float c, float d) {
    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}

constexpr uint32_t PLANE = THREADS * 16;    // 16 bytes for each
constexpr int MOST_SMEM = 200 << 10;
template <int ROW, int BLOCKS = 1>          // planes of a row; blocks that share an SM
constexpr int STAGES = MOST_SMEM / BLOCKS / (ROW * int(PLANE)) < 6 ? MOST_SMEM / BLOCKS / (ROW * int(PLANE)) : 6;

// Two f32 values to an instruction.
struct F2 {
    uint64_t v;
    __device__ __forceinline__ F2() {}
    __device__ __forceinline__ F2(float a, float b) : v(attn::pack2(a, b)) {}
    __device__ __forceinline__ explicit F2(float a) : v(attn::pack2(a, a)) {}
    __device__ __forceinline__ float sum() const {
        float a, b;
        attn::unpack2(v, a, b);
        return a + b;
    }
};
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    a.v = attn::fma2(a.v, b.v, c.v);
    return a;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v));
    return a;
}
__device__ __forceinline__ void pairs(const float (&v)[8], F2 (&p)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = F2(v[2 * j], v[2 * j + 1]);
}
__device__ __forceinline__ void singles(const F2 (&p)[4], float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) attn::unpack2(p[j].v, v[2 * j], v[2 * j + 1]);
}

struct Ring {
    int team, teams;  // threads of a team, teams in the whole grid (a multiple of the classes)
    int classes;
};
// Which rows a team takes: with one group every k.teams-th; else units of rows (group, piece, piece + pieces, ...), of its class.
template <bool GROUPS>
struct Walk;
template <>
struct Walk<false> {
    int64_t offset, d;  // of the row's first element
    int row, n, teams;
    static constexpr int group = 0;
    template <class A>
    __device__ __forceinline__ Walk(const A& g, const Ring& k, int team)
        : offset((int64_t(team) - k.teams) * g.d), d(int64_t(k.teams) * g.d), row(team - k.teams), n(int(g.n)), teams(k.teams) {}
    __device__ __forceinline__ bool next() {
        if (n - row <= teams) return false;
        row += teams, offset += d;
        return true;
    }
};
template <>
struct Walk<true> {
    int64_t offset, d;
    int row, end, unit, group;
    int w, step, per, n, run, pieces, units, cls, classes;  // (there are fewer than 2^31 rows, and no more units)
    template <class A>
    __device__ __forceinline__ Walk(const A& g, const Ring& k, int team)
        : offset(0), d(g.d), row(0), end(0), unit(0), group(0), w(team / k.classes - k.teams / k.classes), step(k.teams / k.classes), n(int(g.n)), run(int(g.gate_rows)), pieces(int(g.pieces)),
          units(int(g.groups * g.pieces)), cls(team % k.classes), classes(k.classes) {
        per = pieces % classes ? 0 : pieces / classes;
    }
    // the next row of the unit, or the first of the team's next one; false: there is none
    __device__ __forceinline__ bool next() {
        if (end - row > pieces) {
            row += pieces, offset += pieces * d;
            return true;
        }
        return next_unit();
    }
    __device__ __forceinline__ bool next_unit() {
        do {
            w += step;
            int piece;
            if (per) {
                group = int(unsigned(w) / unsigned(per)), piece = (w - group * per) * classes;
                if (int64_t(group) * pieces >= units) return false;
                // (classes is a power of two)
                piece += (cls - (group * run + piece)) & (classes - 1);
            } else {  // units of one row
                const int64_t u = int64_t(w) * classes + cls;
                if (u >= units) return false;
                group = int(unsigned(u) / unsigned(run)), piece = int(u) - group * run;
            }
            unit = group * pieces + piece, row = group * run + piece, end = run < n - group * run ? (group + 1) * run : n;
        } while (row >= end);
        offset = row * d;
        return true;
    }
};

// Columns [lo, hi) of a chunk belong to the row.
__device__ __forceinline__ void only(float (&v)[8], int lo, int hi) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j >= lo && j < hi ? v[j] : 0.f;
}
template <class T>
struct Chunks {  // a tensor's chunks (RAGGED: rows that are no whole ones)
    // the chunk that begins with element `at`, a multiple of eight; `left` elements of the tensor are from there on
    static __device__ __forceinline__ void copy(uint32_t to, const T* p, int64_t at, int left) {
#pragma unroll
        for (int q = 0; q < PLANES<T>; ++q) {
            constexpr int EACH = 16 / int(sizeof(T));
            const int here     = max(0, min(EACH, left - q * EACH));
            copy_async(to + q * PLANE, p + at + (here ? q * EACH : 0), here * int(sizeof(T)));
        }
    }
    static __device__ __forceinline__ void copy(uint32_t to, const T* p, int64_t at) {
#pragma unroll
        for (int q = 0; q < PLANES<T>; ++q) copy_async(to + q * PLANE, p + at + q * (16 / int(sizeof(T))), 16);
    }
    // a row's columns of a chunk, zeros for the others
    template <bool RAGGED, class M>
    static __device__ __forceinline__ void get(uint32_t from, F2 (&p)[4], const M& m, int c) {
        Run<T, 8> r;
        float v[8];
        r.a = take16(from);
        if constexpr (PLANES<T> == 2) r.b = take16(from + PLANE);
        r.get(v);
        if (RAGGED ? m.part[c] : !m.any[c]) only(v, m.lo[c], m.hi[c]);
        pairs(v, p);
    }
};
template <bool RAGGED, class T>
__device__ __forceinline__ void put_part(T* p, const float (&v)[8], int lo, int hi) {
    if (!RAGGED || (lo == 0 && hi == 8)) {
        put(p, v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j >= lo && j < hi) put(p + j, *reinterpret_cast<const float(*)[1]>(v + j));
    }
}
// the same where rows are not laid out by chunks (partial sums, a gate's gradient)
template <class T>
__device__ __forceinline__ void put_anywhere(T* p, const float (&v)[8], int lo, int hi) {
    if (lo == 0 && hi == 8 && reinterpret_cast<uintptr_t>(p) % 16 == 0) {
        put(p, v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j >= lo && j < hi) put(p + j, *reinterpret_cast<const float(*)[1]>(v + j));
    }
}
// eight factors from column `at` on, of which those in [lo, hi) are there; zeros for the others
template <class T>
__device__ __forceinline__ void factors_of(const T* p, int lo, int hi, float (&v)[8]) {
    if (lo == 0 && hi == 8 && reinterpret_cast<uintptr_t>(p) % 16 == 0) {
        Run<T, 8> run;
        run.load(p), run.get(v);
    } else {
        Run<T, 1> run[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            run[j].clear();
            if (j >= lo && j < hi) run[j].load(p + j);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) run[j].get(*reinterpret_cast<float(*)[1]>(v + j));
    }
}
__device__ __forceinline__ void factors_part(const Factors& f, int64_t at, int lo, int hi, float (&v)[8]) {
    if (!f.p) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j >= lo && j < hi ? 1.f : 0.f;
    } else if (f.bf16) {
        factors_of(static_cast<const __nv_bfloat16*>(f.p) + at, lo, hi, v);
    } else {
        factors_of(static_cast<const float*>(f.p) + at, lo, hi, v);
    }
}

// Sums over a team of whole warps, in every thread: one barrier, places in turn.
struct Sums {
    float v[2][32][4];
};
__device__ __forceinline__ void meet(int team, int in_block) { asm volatile("bar.sync %0, %1;" ::"r"(in_block + 1), "r"(team) : "memory"); }
__device__ __forceinline__ void ring_sum(float& v, Sums& part, int& turn, int team, int in_block) {
    v = warp_sum(v);
    if (team == 32) return;
    const int warps = team >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) part.v[turn][warp][0] = v;
    meet(team, in_block);
    v = (lane & 15) < warps ? part.v[turn][in_block * warps + (lane & 15)][0] : 0.f;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    turn ^= 1;
}
// Three sums at once. The lanes of a half keep two of four values (the fourth is nothing), those of a quarter one: six exchanges in place of fifteen.
__device__ __forceinline__ void ring_sum(float (&v)[3], Sums& part, int& turn, int team, int in_block) {
    const int lane = threadIdx.x & 31;
    const bool high = lane & 16, odd = lane & 8;
    float a = high ? v[2] : v[0], b = high ? 0.f : v[1];
    a += __shfl_xor_sync(0xffffffffu, high ? v[0] : v[2], 16), b += __shfl_xor_sync(0xffffffffu, high ? v[1] : 0.f, 16);
    float s = odd ? b : a;
    s += __shfl_xor_sync(0xffffffffu, odd ? a : b, 8);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);  // lanes 0, 8, 16: the warp's three sums
    if (team != 32) {
        const int warps = team >> 5, warp = threadIdx.x >> 5, at = lane & 15;
        if ((lane & 7) == 0) part.v[turn][warp][lane >> 3] = s;
        meet(team, in_block);
        const float2 two = at < warps ? *reinterpret_cast<const float2*>(&part.v[turn][in_block * warps + at][high ? 2 : 0]) : make_float2(0.f, 0.f);
        s = (odd ? two.y : two.x) + __shfl_xor_sync(0xffffffffu, odd ? two.x : two.y, 8);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        turn ^= 1;
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) v[i] = __shfl_sync(0xffffffffu, s, i * 8);
}

// A thread's place: its team, and the chunks of a row that are its own.
template <int CH>
struct Mine {
    int team, in_block, t;
    int at[CH], lo[CH], hi[CH];  // first column; of the chunk's eight those that belong to the row, [lo, hi) (none: hi <= lo)
    bool any[CH], part[CH];
    uint32_t place;
    __device__ __forceinline__ Mine(const Ring& k, int64_t d, const uint8_t* smem) {
        in_block = threadIdx.x / k.team, t = threadIdx.x - in_block * k.team;
        const int teams = THREADS / k.team;
        team  = in_block < teams ? int(blockIdx.x) * teams + in_block : k.teams;  // (threads behind the last team: none)
        place = uint32_t(__cvta_generic_to_shared(smem)) + threadIdx.x * 16;
        const int lead = int((team % k.classes) * d & 7);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            at[c] = (c * k.team + t) * 8 - lead;
            lo[c] = max(0, -at[c]), hi[c] = int(min(int64_t(8), d - at[c]));
            any[c] = hi[c] > lo[c], part[c] = lo[c] > 0 || hi[c] < 8;
            if (!any[c]) lo[c] = hi[c] = 0;
        }
    }
};
// The factors of a thread's columns: q = b gate post_gamma, and gamma.
template <int CH>
struct Weights {
    F2 q[CH][4], w[CH][4];
    template <class A>
    __device__ __forceinline__ void load(const A& g, const Mine<CH>& m, int64_t group) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            float post[8], gate[8], gamma[8];
            factors_part(g.post_gamma, m.at[c], m.lo[c], m.hi[c], post), factors_part(g.gate, (g.gate.p ? group * g.d : 0) + m.at[c], m.lo[c], m.hi[c], gate);
            factors_part(g.gamma, m.at[c], m.lo[c], m.hi[c], gamma);
#pragma unroll
            for (int j = 0; j < 8; ++j) post[j] *= g.b * gate[j];
            pairs(post, q[c]), pairs(gamma, w[c]);
        }
    }
};

template <class RT, class HT, int CH, bool RAGGED, bool GROUPS>
__global__ void __launch_bounds__(THREADS, CH == 1 && !GROUPS ? 2 : 1) forward_ring_kernel(const __grid_constant__ Args<RT, HT> g, const __grid_constant__ Ring k) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Sums sums;
    after_previous();
    const Mine<CH> m(k, g.d, smem);
    if (m.team >= k.teams) return;  // (whole teams: their barriers are their own)
    constexpr int PAIR = PLANES<RT> + PLANES<HT>, ROW = CH * PAIR, AHEAD = STAGES<ROW, CH == 1 && !GROUPS ? 2 : 1>;
    Walk<GROUPS> cur(g, k, m.team), ahead = cur;
    const int64_t total = g.n * g.d;
    const float per     = 1.f / float(g.d);
    bool more           = true;
    auto request = [&](uint32_t stage) {
        if (more && (more = ahead.next())) {
            const bool last = ahead.offset + g.d + 8 > total;  // (a chunk may end behind the tensor)
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                if (!m.any[c]) continue;
                const uint32_t to = m.place + stage + c * PAIR * PLANE;
                const int64_t p   = ahead.offset + m.at[c];
                if (RAGGED && last) {
                    const int left = int(min(int64_t(8), total - p));
                    Chunks<RT>::copy(to, g.r, p, left);
                    if (g.h) Chunks<HT>::copy(to + PLANES<RT> * PLANE, g.h, p, left);
                } else {
                    Chunks<RT>::copy(to, g.r, p);
                    if (g.h) Chunks<HT>::copy(to + PLANES<RT> * PLANE, g.h, p);
                }
            }
        }
        copies_end();
    };
    for (int stage = 0; stage < AHEAD; ++stage) request(stage * ROW * PLANE);
    Weights<CH> f;
    int group      = -1;
    uint32_t stage = 0;
    int turn       = 0;
    while (cur.next()) {
        if (cur.group != group) f.load(g, m, group = cur.group);
        copies_wait<AHEAD - 1>();
        F2 v[CH][4], h[CH][4], squares(0.f);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const uint32_t p = m.place + stage + c * PAIR * PLANE;
            Chunks<RT>::template get<RAGGED>(p, v[c], m, c), Chunks<HT>::template get<RAGGED>(p + PLANES<RT> * PLANE, h[c], m, c);
#pragma unroll
            for (int j = 0; j < 4; ++j) squares = fma2(h[c][j], h[c][j], squares);
        }
        float e = 1.f, s = 1.f, sum = squares.sum();
        if (g.post_gamma.p) {
            ring_sum(sum, sums, turn, k.team, m.in_block);
            e = rsqrtf(fmaf(sum, per, g.eps));
        }
        request(stage);
        stage   = stage == (AHEAD - 1) * ROW * PLANE ? 0 : stage + ROW * PLANE;
        squares = F2(0.f);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if (g.h) {
                float out[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[c][j] = fma2(F2(g.a), v[c][j], f.q[c][j] * (h[c][j] * F2(e)));
                singles(v[c], out);
                if (m.any[c]) put_part<RAGGED>(g.r_out + cur.offset + m.at[c], out, m.lo[c], m.hi[c]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) squares = fma2(v[c][j], v[c][j], squares);
        }
        if (g.gamma.p) {
            sum = squares.sum();
            ring_sum(sum, sums, turn, k.team, m.in_block);
            s = rsqrtf(fmaf(sum, per, g.eps));
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                float out[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[c][j] = v[c][j] * (F2(s) * f.w[c][j]);
                singles(v[c], out);
                if (m.any[c]) put_part<RAGGED>(g.x + cur.offset + m.at[c], out, m.lo[c], m.hi[c]);
            }
        }
        if (g.kept && m.t == 0) g.kept[cur.row] = e, g.kept[g.n + cur.row] = s;
    }
}

// GROUPS: the gate has several rows, so that sum D h^ is needed for each unit of rows; else one for all rows will do, from which both dpost_gamma and dgate follow.
template <class RT, class HT, int CH, bool RAGGED, bool GROUPS>
__global__ void __launch_bounds__(THREADS, 1) backward_ring_kernel(const __grid_constant__ Args<RT, HT> g, const __grid_constant__ Ring k) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Sums sums;
    after_previous();
    const Mine<CH> m(k, g.d, smem);
    if (m.team >= k.teams) return;
    constexpr int PAIR = PLANES<RT> + PLANES<HT>, ROW = CH * 2 * PAIR;
    Walk<GROUPS> cur(g, k, m.team), ahead = cur;
    const int64_t total = g.n * g.d;
    const float per     = 1.f / float(g.d);
    // what there is no tensor for stays zero
#pragma unroll 1
    for (int q = 0; q < STAGES<ROW> * ROW; ++q) leave16(m.place + q * PLANE, 0.f, 0.f, 0.f, 0.f);
    bool more = true;
    auto request = [&](uint32_t stage) {
        if (more && (more = ahead.next())) {
            const bool last = ahead.offset + g.d + 8 > total;  // (a chunk may end behind the tensor)
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                if (!m.any[c]) continue;
                const uint32_t to = m.place + stage + c * 2 * PAIR * PLANE;
                const int64_t p   = ahead.offset + m.at[c];
                if (RAGGED && last) {
                    const int left = int(min(int64_t(8), total - p));
                    Chunks<RT>::copy(to, g.r, p, left);
                    if (g.h) Chunks<HT>::copy(to + PLANES<RT> * PLANE, g.h, p, left);
                    if (g.dr_out) Chunks<RT>::copy(to + PAIR * PLANE, g.dr_out, p, left);
                    if (g.dx) Chunks<HT>::copy(to + (PAIR + PLANES<RT>) * PLANE, g.dx, p, left);
                } else {
                    Chunks<RT>::copy(to, g.r, p);
                    if (g.h) Chunks<HT>::copy(to + PLANES<RT> * PLANE, g.h, p);
                    if (g.dr_out) Chunks<RT>::copy(to + PAIR * PLANE, g.dr_out, p);
                    if (g.dx) Chunks<HT>::copy(to + (PAIR + PLANES<RT>) * PLANE, g.dx, p);
                }
            }
        }
        copies_end();
    };
    for (int stage = 0; stage < STAGES<ROW>; ++stage) request(stage * ROW * PLANE);
    F2 dgamma[CH][4], z[CH][4];
    float dpost[GROUPS ? CH : 1][8] = {};
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) dgamma[c][j] = z[c][j] = F2(0.f);
    // the sums of a unit of rows: dgate's, and (as the gate changes) dpost_gamma's
    auto finish = [&](int64_t unit, int64_t group) {
        if constexpr (GROUPS) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                float f[8], w[8], sum[8];
                factors_part(g.post_gamma, m.at[c], m.lo[c], m.hi[c], f), factors_part(g.gate, group * g.d + m.at[c], m.lo[c], m.hi[c], w);
                singles(z[c], sum);
#pragma unroll
                for (int j = 0; j < 8; ++j) dpost[c][j] = fmaf(g.b * w[j], sum[j], dpost[c][j]), f[j] *= g.b * sum[j];
#pragma unroll
                for (int j = 0; j < 4; ++j) z[c][j] = F2(0.f);
                if (!m.any[c]) continue;
                if (g.pieces > 1) put_anywhere(g.part_gate + unit * g.d + m.at[c], f, m.lo[c], m.hi[c]);
                else if (g.gate.bf16) put_anywhere(static_cast<__nv_bfloat16*>(g.dgate) + group * g.d + m.at[c], f, m.lo[c], m.hi[c]);
                else put_anywhere(static_cast<float*>(g.dgate) + group * g.d + m.at[c], f, m.lo[c], m.hi[c]);
            }
        }
    };
    Weights<CH> f;
    int group = -1, unit = -1;
    uint32_t stage = 0;
    int turn       = 0;
    // (a row's e and s are asked for a row ahead)
    float e = 1.f, s = 1.f;
    auto advance = [&] {
        const bool there = cur.next();
        if (there && g.post_gamma.p) e = g.kept[cur.row];
        if (there && g.gamma.p) s = g.kept[g.n + cur.row];
        return there;
    };
    for (bool there = advance(); there;) {
        if constexpr (GROUPS) {
            if (cur.unit != unit && unit >= 0) finish(unit, group);
            unit = cur.unit;
        }
        if (cur.group != group) f.load(g, m, group = cur.group);
        const int64_t offset = cur.offset;
        const F2 e2(e), s2(s);
        const float s1 = s, e1 = e;
        copies_wait<STAGES<ROW> - 1>();
        F2 hat[CH][4], rhat[CH][4], before[CH][4], all[3] = {F2(0.f), F2(0.f), F2(0.f)};
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const uint32_t p = m.place + stage + c * 2 * PAIR * PLANE;
            F2 d[4];
            Chunks<RT>::template get<RAGGED>(p, rhat[c], m, c), Chunks<HT>::template get<RAGGED>(p + PLANES<RT> * PLANE, hat[c], m, c);
            Chunks<RT>::template get<RAGGED>(p + PAIR * PLANE, before[c], m, c), Chunks<HT>::template get<RAGGED>(p + (PAIR + PLANES<RT>) * PLANE, d, m, c);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                hat[c][j]   = hat[c][j] * e2;
                const F2 qh = f.q[c][j] * hat[c][j], t = d[j] * f.w[c][j];
                rhat[c][j]   = s2 * fma2(F2(g.a), rhat[c][j], qh);
                before[c][j] = fma2(s2, t, before[c][j]);
                dgamma[c][j] = fma2(d[j], rhat[c][j], dgamma[c][j]);
                all[0] = fma2(t, rhat[c][j], all[0]), all[1] = fma2(qh, before[c][j], all[1]), all[2] = fma2(qh, rhat[c][j], all[2]);
            }
        }
        there        = advance();
        float sum[3] = {all[0].sum(), all[1].sum(), all[2].sum()};
        ring_sum(sum, sums, turn, k.team, m.in_block);
        request(stage);
        stage = stage == (STAGES<ROW> - 1) * ROW * PLANE ? 0 : stage + ROW * PLANE;
        const float m0 = g.gamma.p ? s1 * sum[0] * per : 0.f, m1 = g.post_gamma.p ? (sum[1] - m0 * sum[2]) * per : 0.f;
        const F2 less(-m0), f1(-m1 * e1);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            F2 dr[4], dh[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const F2 D = fma2(less, rhat[c][j], before[c][j]);
                dr[j]   = F2(g.a) * D;
                z[c][j] = fma2(D, hat[c][j], z[c][j]);
                dh[j]   = fma2(f.q[c][j], D * e2, hat[c][j] * f1);
            }
            if (!m.any[c]) continue;
            float out[8];
            singles(dr, out);
            put_part<RAGGED>(g.dr + offset + m.at[c], out, m.lo[c], m.hi[c]);
            singles(dh, out);
            if (g.dh) put_part<RAGGED>(g.dh + offset + m.at[c], out, m.lo[c], m.hi[c]);
        }
    }
    if constexpr (GROUPS) {
        if (unit >= 0) finish(unit, group);
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        if (!m.any[c]) continue;
        float out[8];
        singles(dgamma[c], out);
        if (g.part_gamma) put_anywhere(g.part_gamma + int64_t(m.team) * g.d + m.at[c], out, m.lo[c], m.hi[c]);
        if constexpr (GROUPS) {
            if (g.part_post) put_anywhere(g.part_post + int64_t(m.team) * g.d + m.at[c], dpost[c], m.lo[c], m.hi[c]);
        } else {
            singles(z[c], out);
            if (g.part_post) put_anywhere(g.part_post + int64_t(m.team) * g.d + m.at[c], out, m.lo[c], m.hi[c]);
        }
    }
}

// out[group, c] = factor[c] times the sum of `count` rows of partial sums, into up to two results; 32 columns a block, every 16th row a warp, 16 of them on their way.
// Bound by the latency of two such reads and a launch: 4.8 MB in 7 us.
struct Result {
    void* out;
    int bf16, times;  // times: by `by` and the factors
    float by;
    Factors factors;
};
struct Join {
    const float* part;
    int64_t groups, count, rows, run;  // a group's units: `count`, or its rows (`run` of them, of `rows` in all), one each
    Result to[2];
};
struct Joins {
    Join j[3];
};
constexpr int JOINED = 512, AT_ONCE = 16;  // threads; rows that each has on their way
__global__ void __launch_bounds__(JOINED) join_kernel(const __grid_constant__ Joins all, int64_t d) {
    __shared__ float sums[JOINED / 32][32];
    after_previous();
    const Join& j   = all.j[blockIdx.z];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = int64_t(blockIdx.x) * 32 + lane;
    for (int64_t group = blockIdx.y; group < j.groups; group += gridDim.y) {
        const float* p      = j.part + group * j.count * d + c;
        const int64_t count = min(j.count, j.rows - group * j.run);
        float v             = 0.f;
        for (int64_t first = warp; first < count; first += AT_ONCE * JOINED / 32) {
            float each[AT_ONCE];
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const int64_t row = first + i * (JOINED / 32);
                each[i]           = c < d && row < count ? p[row * d] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) v += each[i];
        }
        __syncthreads();
        sums[warp][lane] = v;
        __syncthreads();
        if (warp < 2 && c < d && j.to[warp].out) {
            const Result& r = j.to[warp];
            v               = 0.f;
#pragma unroll
            for (int w = 0; w < JOINED / 32; ++w) v += sums[w][lane];
            float one[1] = {1.f};
            if (r.times) factors_at(r.factors, c, one), v *= r.by * one[0];
            if (r.bf16) static_cast<__nv_bfloat16*>(r.out)[group * d + c] = __float2bfloat16(v);
            else static_cast<float*>(r.out)[group * d + c] = v;
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
// Rows of one group: all of them without a gate, and no more than there are.
int64_t group_rows(const Desc& d) {
    const int64_t all = d.n > 0 ? d.n : 1;
    return d.gate && d.gate_rows < all ? d.gate_rows : all;
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
// whether all tensors start on 16 bytes
bool aligned(const Desc& d) {
    bool all = true;
    for (const void* p : {d.r, d.h, d.gamma, d.post_gamma, d.gate, static_cast<const void*>(d.r_out), static_cast<const void*>(d.x), d.dr_out, d.dx, static_cast<const void*>(d.dr),
                          static_cast<const void*>(d.dh), static_cast<const void*>(d.dgate)})
        all = all && aligned16(p);
    return all;
}

// How rows are dealt out: threads and rows of a block, blocks, and units of rows; and what the backward pass leaves for the second launch.
struct Plan {
    bool ring;
    int threads, rows, blocks, columns;  // columns: eights of them that a thread holds (ring)
    Ring k;
    size_t smem;
    int64_t teams, groups, pieces;
    float *gamma, *post, *gate, *z;
    bool shared;
};
Plan plan(const Desc& d, bool backward, bool aligned, Space& space, int sm_count) {
    Plan p{};
    const size_t pair = dtype_size(d.stream_dtype) + dtype_size(d.block_dtype);
    const int64_t run = group_rows(d);
    p.groups          = (d.n + run - 1) / run;
    int classes       = 8;
    while (classes > 1 && d.d % (16 / classes) == 0) classes /= 2;
    // A team's threads hold eight columns each, sixteen where those are too many threads for one team, or (forward, whose columns cost less than what each
    // row costs a thread) for two on an SM. Longer rows, and tensors that do not start on 16 bytes, go without a ring: 8192 x 4096 bf16, one value at a time, in 231 and 538 us.
    const int64_t chunks = (d.d + (classes > 1 ? 7 : 0) + 7) / 8;
    p.columns            = chunks <= (backward ? 512 : 256) ? 1 : 2;
    const int64_t team = up((chunks + p.columns - 1) / p.columns, 32), in_block = team <= THREADS ? THREADS / team : 0;
    const int64_t row  = p.columns * int64_t(PLANE) * int64_t(pair) / 2 * (backward ? 2 : 1);
    p.ring             = aligned && in_block > 0 && row <= MOST_SMEM;
    // Sixteen columns and their sums are more than a thread's registers backward: whole rows are read twice instead where a gate has groups or the stream is F32 (4096 x 8192,
    // one group and four: bf16 155 and 185 us, by a ring 155 and 290; F32 stream 210 and 216, by a ring 240 and 392).
    if (backward && p.columns == 2 && classes == 1 && (p.groups > 1 || d.stream_dtype == MIMK_F32)) p.ring = false;
    if (p.ring) {
        p.k.team = int(team), p.k.classes = classes;
        const int64_t share = !backward && p.columns == 1 && p.groups == 1 ? 2 : 1, stages = MOST_SMEM / share / row;  // blocks to an SM
        p.threads = THREADS, p.smem = size_t(row * (stages < 6 ? stages : 6));
        const int64_t most = int64_t(sm_count) * share * in_block, need = up(d.n, classes);
        p.k.teams = int((need < most ? need : most) / classes * classes);
        p.teams   = p.k.teams;
        p.blocks  = int((p.teams + in_block - 1) / in_block);
        // (no more units than teams, as far as that goes: a team with two of them would be the last)
        p.pieces = p.groups ? p.teams / p.groups / classes * classes : classes;
        if (p.pieces < classes) p.pieces = classes;
    } else if (backward) {
        const int64_t lanes = up((d.d + 7) / (aligned && d.d % 8 == 0 ? 8 : 1), 32), bytes = (p.groups > 1 ? 3 : 2) * up(d.d, 4) * 4;
        p.threads = int(lanes < THREADS ? lanes : THREADS), p.rows = 1;
        p.shared  = bytes <= MOST_SMEM;
        p.smem    = p.shared ? size_t(bytes) : 0;
        const int64_t most = int64_t(sm_count) * (!p.shared ? 1 : bytes <= MOST_SMEM / 4 ? 4 : MOST_SMEM / bytes);
        p.teams = p.blocks = int(d.n < most ? d.n : most);
        p.pieces = p.groups ? (p.teams + p.groups - 1) / p.groups : 1;
    } else {
        const int64_t each = d.d <= 2048 ? 8 : d.d <= 8192 ? 16 : 32, lanes = up((d.d + each - 1) / each, 32);
        p.threads = int(lanes), p.rows = lanes == 32 ? 4 : 1;
        const int64_t need = (d.n + p.rows - 1) / p.rows;
        p.blocks = int(need < (1 << 20) ? need : 1 << 20);
    }
    if (p.pieces > run) p.pieces = run;
    if (!backward) return p;
    auto part = [&](int64_t rows) { return static_cast<float*>(space.take(size_t(rows) * size_t(d.d) * 4)); };
    if (d.gamma) p.gamma = part(p.teams);
    if (d.post_gamma || (d.gate && p.groups == 1)) p.post = part(p.teams);
    if (d.gate && p.pieces > 1 && p.groups > 1) p.gate = part(p.groups * p.pieces);
    if (!p.ring && !p.shared && p.groups > 1) p.z = part(p.teams);
    return p;
}

template <class RT, class HT>
Args<RT, HT> args_of(const Desc& d) {
    Args<RT, HT> g{};
    g.n = d.n, g.d = d.d, g.gate_rows = group_rows(d);
    g.r = static_cast<const RT*>(d.r), g.h = static_cast<const HT*>(d.h);
    g.gamma = {d.gamma, d.gamma_dtype == MIMK_BF16}, g.post_gamma = {d.post_gamma, d.post_gamma_dtype == MIMK_BF16}, g.gate = {d.gate, d.gate_dtype == MIMK_BF16};
    g.r_out = static_cast<RT*>(d.r_out), g.x = static_cast<HT*>(d.x), g.kept = d.kept;
    g.dr_out = static_cast<const RT*>(d.dr_out), g.dx = static_cast<const HT*>(d.dx), g.dr = static_cast<RT*>(d.dr), g.dh = static_cast<HT*>(d.dh);
    g.dgate = d.dgate, g.eps = d.eps, g.a = d.residual_scale, g.b = d.branch_scale;
    return g;
}

template <auto KERN, class A>
int launch_ring(const Plan& p, const A& g, const DeviceInfo& dev, cudaStream_t s) {
    static bool configured[64] = {};
    if (!configured[dev.device & 63]) {
        MIMK_CUDA_TRY(cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_SMEM));
        configured[dev.device & 63] = true;
    }
    return launch_after(KERN, unsigned(p.blocks), unsigned(p.threads), p.smem, s, g, p.k);
}
template <int V>
struct Number {
    static constexpr int value = V;
};
// f(columns, whether rows are no whole chunks, whether the gate has several rows)
template <class F>
int with_columns(const Plan& p, F&& f) {
    const auto rest = [&](auto columns) {
        if (p.k.classes > 1) return p.groups > 1 ? f(columns, Number<1>(), Number<1>()) : f(columns, Number<1>(), Number<0>());
        return p.groups > 1 ? f(columns, Number<0>(), Number<1>()) : f(columns, Number<0>(), Number<0>());
    };
    return p.columns == 1 ? rest(Number<1>()) : rest(Number<2>());
}
template <class... P, class... A>
int launch(void (*kern)(P...), dim3 grid, dim3 block, cudaStream_t s, A&&... args) {
    cudaLaunchAttribute early = {};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization, early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = grid, config.blockDim = block, config.stream = s, config.attrs = &early, config.numAttrs = 1;
    return note_cuda_error(cudaLaunchKernelEx(&config, kern, static_cast<A&&>(args)...));
}

template <class RT, class HT, int VEC>
int forward(const Desc& d, const Plan& p, const DeviceInfo& dev, cudaStream_t s) {
    Args<RT, HT> g = args_of<RT, HT>(d);
    g.groups = p.groups, g.pieces = p.pieces;
    if (p.ring) return with_columns(p, [&](auto columns, auto ragged, auto several) { return launch_ring<forward_ring_kernel<RT, HT, columns.value, ragged.value, several.value>>(p, g, dev, s); });
    auto kern = forward_kernel<RT, HT, VEC, 32 / VEC, 1024>;
    if constexpr (VEC == 1) {  // (whole rows of up to 8192 columns are planned with a ring)
        if (d.d <= 8192) kern = d.d <= 2048 ? forward_kernel<RT, HT, 1, 8, 256> : forward_kernel<RT, HT, 1, 16, 512>;
    }
    return launch(kern, dim3(unsigned(p.blocks)), dim3(p.threads, p.rows), s, g);
}
template <class RT, class HT, int VEC>
int backward(const Desc& d, const Plan& p, const DeviceInfo& dev, cudaStream_t s) {
    Args<RT, HT> g = args_of<RT, HT>(d);
    g.part_gamma = p.gamma, g.part_post = p.post, g.part_gate = p.gate, g.part_z = p.z, g.shared = p.shared, g.groups = p.groups, g.pieces = p.pieces;
    const bool several = p.groups > 1;
    if (p.ring) {
        MIMK_TRY(with_columns(p, [&](auto columns, auto ragged, auto several) {
            if constexpr (columns.value == 2 && !ragged.value && (several.value || sizeof(RT) == 4)) return int(MIMK_E_UNSUPPORTED);  // (planned without a ring)
            else return launch_ring<backward_ring_kernel<RT, HT, columns.value, ragged.value, several.value>>(p, g, dev, s);
        }));
    } else {
        static bool configured[64] = {};
        if (!configured[dev.device & 63]) {
            MIMK_CUDA_TRY(cudaFuncSetAttribute(backward_kernel<RT, HT, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_SMEM));
            configured[dev.device & 63] = true;
        }
        MIMK_TRY(launch_after(backward_kernel<RT, HT, VEC>, unsigned(p.blocks), unsigned(p.threads), p.smem, s, g));
    }
    Joins all{};
    int count    = 0;
    int64_t most = 1;
    if (p.gamma) all.j[count++] = {p.gamma, 1, p.teams, p.teams, 0, {{d.dgamma, d.gamma_dtype == MIMK_BF16}}};
    if (p.post && !several) {
        all.j[count++] = {p.post, 1, p.teams, p.teams, 0, {{d.post_gamma ? d.dpost_gamma : nullptr, d.post_gamma_dtype == MIMK_BF16, 1, g.b, g.gate}, {d.gate ? d.dgate : nullptr, d.gate_dtype == MIMK_BF16, 1, g.b, g.post_gamma}}};
    } else if (p.post) {
        all.j[count++] = {p.post, 1, p.teams, p.teams, 0, {{d.dpost_gamma, d.post_gamma_dtype == MIMK_BF16}}};
    }
    if (p.gate) all.j[count++] = {p.gate, p.groups, p.pieces, d.n, g.gate_rows, {{d.dgate, d.gate_dtype == MIMK_BF16}}}, most = p.groups;
    if (!count) return MIMK_OK;
    return launch(join_kernel, dim3(unsigned((d.d + 31) / 32), unsigned(most < 65535 ? most : 65535), unsigned(count)), dim3(JOINED), s, all, d.d);
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
    const bool whole = aligned(*d);
    const Plan p     = plan(*d, false, whole, space, dev->sm_count);
    return whole && d->d % 8 == 0 ? MIMK_BY_TYPES(forward, 8, *d, p, *dev, s) : MIMK_BY_TYPES(forward, 1, *d, p, *dev, s);
}

extern "C" int mimk_residual_rmsnorm_workspace(const mimk_residual_rmsnorm_desc* d, uint64_t* bytes) {
    MIMK_TRY(check(d));
    if (!bytes) return MIMK_E_ARG;
    int st                = MIMK_OK;
    const DeviceInfo* dev = device_info(&st);
    if (!dev) return st;
    Space space(nullptr);
    *bytes = 0;
    if (!d->n || !d->d) return MIMK_OK;
    // (whatever the tensors' addresses turn out to be)
    plan(*d, true, true, space, dev->sm_count);
    Space other(nullptr);
    plan(*d, true, false, other, dev->sm_count);
    *bytes = space.used() > other.used() ? space.used() : other.used();
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
    const bool whole = aligned(*d);
    const Plan p     = plan(*d, true, whole, space, dev->sm_count);
    if (space.used() > d->workspace_bytes || (space.used() && !d->workspace)) return MIMK_E_WORKSPACE;
    if (space.used() && !aligned16(d->workspace)) return MIMK_E_ALIGN;
    return whole && d->d % 8 == 0 ? MIMK_BY_TYPES(backward, 8, *d, p, *dev, s) : MIMK_BY_TYPES(backward, 1, *d, p, *dev, s);
}
