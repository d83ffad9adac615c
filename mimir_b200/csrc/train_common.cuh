// What the operators of a training step share: their workspace, matrices laid out for TMA, and how the k-blocks of few tiles are dealt out.
#pragma once

#include "gemm_group.cuh"

namespace mimk {

// Pieces of a caller's buffer, 256 bytes apart. Without a buffer it only counts, so that one plan gives a call its pieces and a size query
// its answer.
class Space {
  public:
    explicit Space(void* base) : base_(static_cast<uint8_t*>(base)) {}
    void* take(size_t bytes) {
        const size_t at = used_;
        used_ += (bytes + 255) & ~size_t(255);
        return base_ ? base_ + at : nullptr;
    }
    size_t used() const { return used_; }

  private:
    uint8_t* base_;
    size_t used_ = 0;
};

inline int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// A bf16 matrix that TMA can read (or write): the caller's own, or one in the workspace whose rows are padded to whole 16 bytes.
struct Staged {
    group::Mat own{}, use{};
    bool copied() const { return own.p != use.p || own.pitch != use.pitch; }
};
inline Staged stage(Space& space, const void* p, int64_t rows, int64_t cols) {
    Staged s;
    s.own = s.use = {p, rows, cols, cols};
    if (!group::tma_can_read(p, cols)) {
        s.use.pitch = up(cols, 8);
        s.use.p     = space.take(size_t(rows) * size_t(s.use.pitch) * 2);
        if (!s.use.p) s.use.p = reinterpret_cast<const void*>(uintptr_t(256));  // (counting only)
    }
    return s;
}
// rows x cols bf16 from one pitch to another
int copy_rows(const void* from, int64_t from_pitch, void* to, int64_t to_pitch, int64_t rows, int64_t cols, cudaStream_t s);
inline int stage_in(const Staged& x, cudaStream_t s) {
    return x.copied() ? copy_rows(x.own.p, x.own.pitch, const_cast<void*>(x.use.p), x.use.pitch, x.own.rows, x.own.cols, s) : MIMK_OK;
}
inline int stage_out(const Staged& x, cudaStream_t s) {
    return x.copied() ? copy_rows(x.use.p, x.use.pitch, const_cast<void*>(x.own.p), x.own.pitch, x.own.rows, x.own.cols, s) : MIMK_OK;
}

// How many tiles share the k-blocks of one: the number that ends first, counting rounds of tiles over the pairs of SMs, 6 k-blocks' time
// for a tile's ends, the f32 partial results written and read (0.27 us a k-block), and the launch that adds them up. The gated block forward and
// backward, with this rule and with one number for both products: 64 rows, 4096 x 14336 x 4096: 281 us; 431 (one), 333 (two), 297 (three),
// 283 (four), 287 (eight), 295 (sixteen). 300 rows, 1000 x 3000 x 1000: 73.5; 110, 91, 82, 78, 74 (eight). 1777 rows, 1024 x 2816 x 1024: 122; 128, 124, 126, 133,
// 151 (eight).
int pick_splits(int64_t m, int64_t n, int64_t kblocks, int sm_count);
// out[r, c] = sum_s part[s][r][c] as bf16; part: `splits` f32 matrices of `rows_pad` rows of `part_pitch`
int sum_parts(const float* part, int splits, int64_t rows_pad, int64_t part_pitch, void* out, int64_t out_pitch, int64_t rows, int64_t cols, cudaStream_t s);

}  // namespace mimk
