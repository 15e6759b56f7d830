// Decode attention of requests with different lengths over one page pool.
//
//   o[b, h] = sum_t w_t v_t / sum_t w_t,  w_t = exp(scale q[b, h] . k_t),
//   t in [start_b, len_b), k_t and v_t rows of kv head h / (Hq / Hkv)
//
// in one pass over K and V with a running maximum of q . k and sum.  A weight is the power of
// scale * (q . k - maximum), the difference taken first: the maximum's own exponent is then exact
// however large the logits are, where the difference of two rounded products is off by up to half a
// step of the larger (32 at 1e9, beyond what a weight can hold).
//
// Work is cut into units of TT tokens of one (request, kv head, group of query heads): a
// segment is all units of one such triple, and the units of all segments in a row are dealt out
// to the CTAs, and within a CTA to its warps, in equal contiguous runs.  So a long request is
// split over many warps and short ones share one, whatever the lengths are; they are only known
// on the device, and every CTA sums the unit counts of all requests itself.
//
// A warp writes the outputs of the segments that lie within its run.  At either end of the run
// there may be a part of a segment, of which it keeps (maximum, sum, accumulator).  The parts
// of a CTA are joined in shared memory when its warps are done, which leaves at most one part
// at either end of the CTA's run; those go to the workspace, and merge_kernel joins them.  Parts
// are joined in the order of the tokens, so results do not depend on timing, and nothing in the
// workspace has to be set before the call.
#include <float.h>
#include <math.h>

#include <atomic>

#include "rkv_common.cuh"
#include "rkv_kernels.h"
#include "rkv_ragged.h"
#include "rkv_sm100.cuh"

namespace rkv {
namespace ragged {

static __device__ int g_error;

constexpr int kCtas = 148;      // one persistent CTA per SM
constexpr int kMostWarps = 8;   // warps per CTA of any kernel here
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Natural logarithm of sum * exp(scale * top) / 2^bias.  The hardware's log2 is off by at most 2^-22
// (absolutely, or relatively to a result above one), as much as the hardware's 2^x in the sum itself.
__device__ __forceinline__ float lse_of(const DecodeParams& p, float top, float sum) {
    return fmaf(top, p.scale, (__log2f(sum) - p.bias) * kLn2);
}

// First and last token of request b, clamped to the page table's capacity.
__device__ __forceinline__ void range_of(const DecodeParams& p, int b, int64_t* first, int64_t* last) {
    const int64_t capacity = p.W * p.P;
    int64_t n = p.lengths[b], s = p.starts ? p.starts[b] : 0;
    if (n < 0 || n > capacity || s < 0) {
        atomicMax(&g_error, kErrLength);
        n = min(max(n, (int64_t)0), capacity);
        s = max(s, (int64_t)0);
    }
    *first = min(s, capacity);
    *last = n;
}

// Tiles of a request: those that hold tokens of [first, last), and one (empty) where none does.
template <int TT>
__device__ __forceinline__ int64_t tiles_of(int64_t first, int64_t last) {
    return last > first ? (last + TT - 1) / TT - first / TT : 1;
}

// What a segment costs besides its tiles, in tiles: its queries, its outputs, the change of
// pages.  Runs are of equal cost, so a segment of n tiles has n + over_of(TT) units, the first of
// which hold no tile.  With 1, 2 and 3 of them, tiles of 16 (16 heads on each of 2 x 128): 64 requests
// of up to 3000 tokens 22.4, 20.3 and 20.1 us, 8 of 18310 39.2, 37.7 and 38.6; tiles of 32: 64 of up to
// 4093 (8 heads x 128) 34.5, 34.0 and 33.9, 255 of up to 509 (16 x 64) 24.2, 25.8 and 27.4.
__host__ __device__ constexpr int over_of(int tile_tokens) { return tile_tokens <= 16 ? 2 : 1; }

// Segments of so few tiles are not split between warps, or between CTAs: the boundary between two
// runs moves to the nearer end of its segment.  Where no segment can have more tiles than are
// split between CTAs, merge_kernel is not launched.
// With at least half as many segments as warps, moving boundaries costs less balance than parts
// cost joins: 64 requests of 250 tokens (8 kv heads x 128, 8 tiles) take 15.7 us whole and 23.1
// split, 64 of 500 28.8 and 34.8; limits of 12 and 16 tiles for warps cost requests of mixed
// lengths more than they gave (255 of 0 to 509 tokens, 16 heads x 64: 24.2 us, 26.6 and 26.8).
// With fewer, a segment has a CTA to itself if `most`, the tiles that the page table has room for,
// are at most two per warp: 8 requests of 250 tokens (8 heads x 128) take 8.6 us, 10.3 with a limit
// of four tiles for both, 1 of 77 6.6 and 7.2, 1 of 256 8.3 and 9.6.  Up to four tiles per warp, 1
// of 500 takes 10.9 us instead of 9.3; split between warps from two tiles on, not three, 1 of 64
// takes 6.8 us instead of 6.1.  Where other segments may be longer, this keeps a CTA at what all
// could share (5 requests of up to 9001 tokens in fp32, 4 heads x 64, windows of 1 to 5000: 11.9 us
// instead of 10.7).
struct Whole {
    int warp, cta;
};
constexpr int kWarpShort = 2, kShortPerWarp = 2, kWarpFew = 4, kWarpMany = 8, kCtaMany = 16;
constexpr Whole whole_tiles(int64_t segments, int64_t most, int warps_per_cta) {
    if (2 * segments >= kCtas * warps_per_cta) return Whole{kWarpMany, kCtaMany};
    if (most <= kShortPerWarp * warps_per_cta) return Whole{kWarpShort, kShortPerWarp * warps_per_cta};
    return Whole{kWarpFew, kWarpFew};
}

// a / b of non-negative numbers
__device__ __forceinline__ int divide(int a, int b) { return (int)((uint32_t)a / (uint32_t)b); }
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) { return a / b; }

// n runs of as nearly equal length as may be, the longer ones first: with q = units / n and
// x = units % n, run i starts at i q + min(i, x).
template <typename I>
struct Deal {
    I q, x;
    __device__ __forceinline__ Deal(I units, I n) {
        q = divide(units, n);
        x = units - q * n;
    }
    __device__ __forceinline__ I start(I i) const { return i * q + min(i, x); }
    // the run that holds a unit
    __device__ __forceinline__ I of(I unit) const {
        const I longer = x * (q + 1);
        return unit < longer ? divide(unit, q + 1) : x + divide(unit - longer, q);
    }
};

// A part of a segment in memory: HG x {maximum, sum}, then HG rows of D accumulators, D + 4
// floats apart (in shared memory, the 8 rows x 4 columns that a warp writes at a time then lie
// in different banks).
struct Part {
    float* at; int HG, D;
    __device__ float& top(int row) const { return at[2 * row]; }
    __device__ float& sum(int row) const { return at[2 * row + 1]; }
    __device__ float* acc(int row) const { return at + 2 * HG + row * (D + 4); }
    __host__ __device__ static constexpr int floats(int hg, int d) { return hg * (d + 6); }
};

// Workspace: for each CTA what the part at the end of its run belongs to, then two parts per
// CTA (of a segment that began before its run; of one that began in it and goes on), then one
// per warp (of a segment that began before the warp's run and ended in it).
struct Workspace {
    int4* open; float* base; int64_t stride; int HG, D;
    __host__ __device__ static int64_t bytes(int64_t warps, int64_t HG, int64_t D) {
        return kCtas * 16 + (2 + warps) * kCtas * Part::floats((int)HG, (int)D) * 4;
    }
    __device__ Workspace(const DecodeParams& p, int hg)
        : open(static_cast<int4*>(p.ws)), base(reinterpret_cast<float*>(open + kCtas)),
          stride(Part::floats(hg, p.D)), HG(hg), D(p.D) {}
    __device__ Part cta(int c, int which) const { return Part{base + (2 * c + which) * stride, HG, D}; }
    __device__ Part warp(int64_t worker) const { return Part{base + (2 * kCtas + worker) * stride, HG, D}; }
};

// The runs of a CTA and of a warp in it.
struct Runs {
    int64_t total;          // units of all requests
    int64_t ctas;           // CTAs that have a run (a unit per warp at least)
    int64_t cta1;           // end of the CTA's run
    int64_t count;          // tiles of the warp's run
    int b, seg;             // its first tile: request, segment of the request, tile of the segment
    int64_t tile, tiles, first, last;   // and the request's tiles per segment, and its tokens
};

// Unit counts are 31-bit numbers wherever the page tables cannot hold more (p.narrow): this code
// runs once and takes as long as it has instructions.
template <typename I, int TT, int NW>
__device__ __forceinline__ Runs find_runs_in(const DecodeParams& p, I per_tile, Whole whole, I* s_sums, I* s_before) {
    constexpr int T = NW * 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (p.B + T - 1) / T;
    const int b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
    I mine = 0;
    int64_t f = 0, l = 0;
    bool between = false;       // a segment that may be split between warps, but not between CTAs
#pragma unroll 1
    for (int b = b0; b < b1; ++b) {
        range_of(p, b, &f, &l);
        const I t = (I)tiles_of<TT>(f, l);
        mine += (t + over_of(TT)) * per_tile;
        between = between || (t > whole.warp && t <= whole.cta);
    }
    I x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const I y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) s_sums[warp] = x;
    __syncthreads();
    constexpr int kOver = over_of(TT);
    Runs r{};
    I before = x - mine, total = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        const I y = s_sums[w];
        before += w < warp ? y : 0;
        total += y;
    }
    s_before[tid] = before;
    between = __syncthreads_or(between);
    const I ctas = max((I)1, min((I)gridDim.x, divide(total, (I)NW)));
    r.total = total;
    r.ctas = ctas;
    if ((I)blockIdx.x >= ctas) return r;
    // Of each boundary: the first tile behind it, the tiles before that one, and the unit at which
    // the boundary has come to lie.  Even lanes look for the start of a run, odd ones for its end;
    // first of the CTA's run (if its boundaries may move where warps' do not), then of the warp's
    // share of it.
    const Deal<I> deal(total, ctas);
    I target = deal.start((I)blockIdx.x + (lane & 1)), tiles_before = 0, tiles = 0, tile = 0;
    int b = 0;
#pragma unroll 1
    for (int pass = between ? 0 : 1; pass < 2; ++pass) {
        if (pass == 1) {
            const I cta0 = __shfl_sync(0xffffffffu, target, 0), cta1 = __shfl_sync(0xffffffffu, target, 1);
            r.cta1 = cta1;
            target = cta0 + Deal<I>(cta1 - cta0, NW).start(warp + (lane & 1));
        }
        const int upto = pass == 0 ? whole.cta : whole.warp;
        if (target >= total) {
            tiles_before = total - kOver * per_tile * p.B;
            continue;
        }
        int i = 0;
#pragma unroll
        for (int step = 512; step > 0; step >>= 1)
            if (i + step < T && s_before[i + step] <= target) i += step;
        I at = s_before[i];
        b = i * per;
        range_of(p, b, &f, &l);
        tiles = (I)tiles_of<TT>(f, l);
        I units = (tiles + kOver) * per_tile;
#pragma unroll 1
        while (target >= at + units) {      // (only where a thread has summed several requests)
            at += units;
            range_of(p, ++b, &f, &l);
            tiles = (I)tiles_of<TT>(f, l);
            units = (tiles + kOver) * per_tile;
        }
        const I length = tiles + kOver;
        r.seg = (int)divide(target - at, length);
        const I seg_at = at + r.seg * length, in_seg = target - seg_at;
        tile = max((I)0, in_seg - kOver);
        if (tiles <= upto) {
            tile = 2 * in_seg > length ? tiles : 0;
            target = seg_at + (tile ? length : 0);
        }
        tiles_before = at - kOver * per_tile * b + r.seg * tiles + tile;
        if (tile == tiles) {        // the start of the next segment
            tile = 0;
            if (++r.seg == per_tile) {
                r.seg = 0;
                if (++b < p.B) {
                    range_of(p, b, &f, &l);
                    tiles = (I)tiles_of<TT>(f, l);
                }
            }
        }
    }
    r.count = __shfl_sync(0xffffffffu, tiles_before, 1) - __shfl_sync(0xffffffffu, tiles_before, 0);
    r.b = __shfl_sync(0xffffffffu, b, 0);
    r.seg = __shfl_sync(0xffffffffu, r.seg, 0);
    r.tile = __shfl_sync(0xffffffffu, tile, 0);
    r.tiles = __shfl_sync(0xffffffffu, tiles, 0);
    r.first = __shfl_sync(0xffffffffu, f, 0);
    r.last = __shfl_sync(0xffffffffu, l, 0);
    return r;
}

template <int TT, int NW>
__device__ __forceinline__ Runs find_runs(const DecodeParams& p, int groups, Whole whole) {
    __shared__ int64_t s_sums[NW], s_before[NW * 32];
    const int per_tile = p.Hkv * groups;
    if (p.narrow)
        return find_runs_in<int, TT, NW>(p, per_tile, whole, reinterpret_cast<int*>(s_sums), reinterpret_cast<int*>(s_before));
    return find_runs_in<int64_t, TT, NW>(p, per_tile, whole, s_sums, s_before);
}

// What a warp leaves for the join: the part of a segment that began before its run (`head`), and
// of one that began in its run and goes on behind it (`tail`).  Of the warp's two places in shared
// memory, a part that is there at the end of the run is in the first, and a head that ended
// before (`early`) in the second.
struct Left {
    int head, ends, early, head_b, head_seg;
    int tail, tail_b, tail_seg;
    int64_t rest;           // tiles of the last segment behind the run
};

constexpr int kJoinRows = 2;

// What a part of maximum `top` weighs where `most` is the largest.  Never zero: an infinity of V in
// a part stays one, however little the part weighs.
__device__ __forceinline__ float part_weight(const DecodeParams& p, float top, float most) {
    return fmaxf(sm100::ex2((top - (most == -INFINITY ? 0.f : most)) * (p.scale * kLog2e)), FLT_MIN);
}

__device__ __forceinline__ float4 lds_float4(uint32_t at, bool on) {
    float4 v;
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %5, 0;\n\tmov.f32 %0, 0f00000000;\n\t"
                 "mov.f32 %1, 0f00000000;\n\tmov.f32 %2, 0f00000000;\n\tmov.f32 %3, 0f00000000;\n\t"
                 "@q ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];\n\t}"
                 : "=&f"(v.x), "=&f"(v.y), "=&f"(v.z), "=&f"(v.w)
                 : "r"(at), "r"((uint32_t)on)
                 : "memory");
    return v;
}

// Joins the parts of a CTA's warps.  In the order of the warps, a tail, or the first head, starts
// a chain, the heads behind it belong to the same segment, and one that ends closes it.  A warp
// takes kJoinRows rows of a chain at a time: lane 8 y + v weighs row y of the part of warp v, and
// the lanes add the rows up, four elements each.
// parts: two places of `place` floats per warp, `stride` floats apart.
template <int NW, int HG, int DT>
__device__ __forceinline__ void join_parts(const DecodeParams& p, const Runs& r, const Workspace& ws,
                                           const Left* left, float* parts, int stride, int place, int groups) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int G = p.Hq / p.Hkv;
    const int c = blockIdx.x;
    static_assert(NW <= 8 && HG % kJoinRows == 0, "lanes of a task");
    const bool in = lane < NW;
    const unsigned heads = __ballot_sync(0xffffffffu, in && left[lane].head);
    const unsigned tails = __ballot_sync(0xffffffffu, in && left[lane].tail);
    const unsigned closing = __ballot_sync(0xffffffffu, in && left[lane].head && left[lane].ends);
    const unsigned early = __ballot_sync(0xffffffffu, in && left[lane].early);
    if (threadIdx.x == 0) ws.open[c] = make_int4(-1, 0, 0, 0);
    int turn = warp;    // rows are dealt to the warps over all chains
    // chain 0: the first head; chain w + 1: the tail of warp w
    unsigned todo = tails << 1 | (heads & 1);
#pragma unroll 1
    while (todo) {
        const int i = __ffs(todo) - 1;
        todo &= todo - 1;
        const int w = i == 0 ? 0 : i - 1;
        const unsigned behind = 0xfffffffeu << w;
        const unsigned closers = i == 0 && (closing & 1) ? 1u : closing & behind;
        const bool closed = closers != 0;
        const unsigned upto = closed ? (closers & -closers) * 2 - 1 : 0xffffffffu;
        const unsigned members = (heads & behind & upto) | 1u << w;
        const unsigned second = i == 0 ? early : early & behind;
        const int b = i ? left[w].tail_b : left[w].head_b;
        const int seg = i ? left[w].tail_seg : left[w].head_seg;
        const int h = groups == 1 ? seg : seg / groups, gi = groups == 1 ? 0 : seg % groups;
        const int hq0 = h * G + gi * HG, ng = min(HG, G - gi * HG);
        const bool whole = i > 0 && closed;
        const Part to = ws.cta(c, i > 0);
        constexpr int R = kJoinRows;
        int task = turn;
#pragma unroll 1
        for (; task * R < ng; task += NW) {
            const int row0 = task * R, v = lane & 7;
            const bool mine = members >> v & 1;
            const int own_row = row0 + (R == 1 ? 0 : lane >> 3 & (R - 1));
            const Part own{parts + (mine ? v : w) * stride + (mine && second >> v & 1 ? place : 0), HG, p.D};
            const float t = mine ? own.top(own_row) : -INFINITY;
            float top = t, sum = mine ? own.sum(own_row) : 0.f;
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float weight = mine ? part_weight(p, t, top) : 0.f;
            if (mine) sum *= weight;
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (v == 0 && lane < 8 * R && own_row < ng) {
                if (!whole) { to.top(own_row) = top; to.sum(own_row) = sum; }
                else if (p.lse) p.lse[(int64_t)b * p.Hq + hq0 + own_row] = lse_of(p, top, sum);
            }
            const float inverse = !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
            const uint32_t from = sm100::smem_u32(Part{parts, HG, p.D}.acc(row0));
#pragma unroll 1
            for (int d = lane * 4; d - lane * 4 < p.D; d += 128) {
                float o[R][4];
#pragma unroll
                for (int y = 0; y < R; ++y)
#pragma unroll
                    for (int x = 0; x < 4; ++x) o[y][x] = 0.f;
                if (p.D % 4 == 0) {
#pragma unroll
                    for (int u = 0; u < NW; ++u) {
                        const bool on = (members >> u & 1) && d < p.D;
                        const uint32_t at = from + (u * stride + (second >> u & 1 ? place : 0) + d) * 4;
#pragma unroll
                        for (int y = 0; y < R; ++y) {
                            const float a = __shfl_sync(0xffffffffu, weight, y * 8 + u);
                            const float4 f = lds_float4(at + y * (p.D + 4) * 4, on);
                            o[y][0] = fmaf(f.x, a, o[y][0]); o[y][1] = fmaf(f.y, a, o[y][1]);
                            o[y][2] = fmaf(f.z, a, o[y][2]); o[y][3] = fmaf(f.w, a, o[y][3]);
                        }
                    }
                } else {
#pragma unroll 1
                    for (int u = 0; u < NW; ++u) {
                        const Part part{parts + u * stride + (second >> u & 1 ? place : 0), HG, p.D};
#pragma unroll
                        for (int y = 0; y < R; ++y) {
                            const float a = __shfl_sync(0xffffffffu, weight, y * 8 + u);
                            if (!(members >> u & 1)) continue;
#pragma unroll
                            for (int x = 0; x < 4; ++x)
                                if (d + x < p.D) o[y][x] = fmaf(part.acc(row0 + y)[d + x], a, o[y][x]);
                        }
                    }
                }
#pragma unroll
                for (int y = 0; y < R; ++y) {
                    const int row = row0 + y;
                    const float scale = __shfl_sync(0xffffffffu, inverse, y * 8);
                    if (row >= ng) break;
                    const int64_t at = (int64_t)b * p.o_stride_b + (int64_t)(hq0 + row) * p.o_stride_h + d;
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        if (d + x >= p.D) break;
                        if (whole) store_elt(p.out, at + x, DT < 0 ? p.dtype : DT, o[y][x] * scale);
                        else to.acc(row)[d + x] = o[y][x];
                    }
                }
            }
        }
        turn = task - (ng + R - 1) / R;
        turn = turn >= NW ? turn - NW : turn;
        if (i > 0 && !closed && threadIdx.x == 0) {
            const int z = 31 - __clz(members);      // last warp of the chain
            const int64_t last = r.cta1 + left[z].rest - 1;
            ws.open[c] = make_int4(b, seg, (int)(Deal<int64_t>(r.total, r.ctas).of(last) - c), 0);
        }
    }
}

// Position in the row of tiles: request, kv head, group of query heads, tile.
template <int TT>
struct Walk {
    int b, h, gi, tile, tiles, first, last;
    __device__ __forceinline__ void start(const Runs& r, int groups) {
        b = r.b;
        h = groups == 1 ? r.seg : r.seg / groups;
        gi = r.seg - h * groups;
        tile = (int)r.tile;
        tiles = (int)r.tiles;
        first = (int)r.first;
        last = (int)r.last;
    }
    __device__ __forceinline__ void next(const DecodeParams& p, int groups) {
        if (++tile < tiles) return;
        tile = 0;
        if (++gi < groups) return;
        gi = 0;
        if (++h < p.Hkv) return;
        h = 0;
        if (++b >= p.B) return;
        int64_t f, l;
        range_of(p, b, &f, &l);
        first = (int)f;
        last = (int)l;
        tiles = (int)tiles_of<TT>(f, l);
    }
    __device__ __forceinline__ int token0() const { return ((uint32_t)first / TT + tile) * TT; }
};

// ------------------------------------------------------------------------------------------
// 16-bit types, on tensor cores.  One warp works alone: it copies its tiles (TT tokens of K and
// V) into a ring of STAGES buffers of its own with 16-byte asynchronous copies, row by row
// through the page table, and multiplies with m16n8k16 from there, tokens and dims in the rows
// and NH x 8 query heads in the columns:
//   S^T = K Q^T  (16 tokens x 8 heads),    O^T += V^T P^T  (16 dims x 8 heads).
// With the heads in the narrow dimension no product is spent on padding up to 16 rows, and O
// takes half the registers.  P^T gets from the accumulator's layout to the operand's by an 8x8
// transpose in registers.
// Rounding P to 16 bits alone would add an error as large as the output's own rounding, so P
// goes in as hi + lo, both 16-bit (with 16 heads, where products cost most, 19.6 us instead of
// 19.4 for 16 requests of up to 16384 tokens, 37.7 and 37.2 for 8 of 18310).  The base of the power
// is a maximum seen so far that is only renewed when a logit exceeds it by more than kSlack (in
// exponents of two), which saves the reduction over lanes on most tiles; weights are then at most
// 2^kSlack instead of 1.  In fp16 they are scaled by 2^kBias besides, so that small ones stay in
// fp16's normal range; that scale is taken out of the log-sum-exp and cancels in the output.
// Rows outside the request's range are filled with zeros without being read: what the pool
// holds there (NaN included) never enters a product.
// Bound by memory: 8 requests of 32768 tokens (8 x 128, bf16) take 181 us, 5.9 TB/s of K and V,
// 1 of 131072 (4 x 128) 53 us, 5.1 TB/s; about 7 us of a call are not: its launches, the sums over
// the requests, the first tile's way, the joins.  Tensor pipes are active an eighth of the time with
// 7 heads per kv head; 16 heads reach 4.0 TB/s (8 requests of 18310 tokens, 2 x 128).
// ------------------------------------------------------------------------------------------
// 16 bytes, or zeros without a read
__device__ __forceinline__ void copy16_or_zero(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <bool kBf16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    if constexpr (kBf16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}
template <bool kBf16>
__device__ __forceinline__ float2 unpack16(uint32_t x) {
    if constexpr (kBf16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
    else return __half22float2(*reinterpret_cast<const __half2*>(&x));
}

template <int DP, int NH, int TT, int NW, int STAGES>
struct TcShape {
    static constexpr int kPitch = DP * 2 + 16;          // odd in 16-byte units: no bank conflicts
    static constexpr int kPlane = TT * kPitch;          // K or V of a tile
    static constexpr int kStage = 2 * kPlane + NH * 8 * kPitch;     // and the queries of its segment
    static constexpr int kSmem = NW * STAGES * kStage;
};

constexpr float kSlack = 8.f;
constexpr float tc_bias(bool bf16) { return bf16 ? 0.f : 6.f; }

// Sums of the infinite and NaN elements of V over the tokens [t0, t1) of a request, for dims
// 8 i + lane / 4 (zero where a column has none): what such a column of the output is, whatever the
// (positive) weights are.  The products give NaN for it, since the low half of a weight may be zero
// or negative.  Read again from the pool, by calls of such values only (the check costs 0.1 to 0.4 us
// of a call: one short request 6.4 and 6.6, 64 of 500 tokens, 16 heads on each of 2 x 128, 20.9 and
// 21.3).  The four lanes of a dim share the tokens.
template <bool kBf16, int DP>
__device__ __noinline__ void odd_columns(float (&sum)[DP / 8], const void* v, const int64_t* table, int64_t num_slots,
                                         int64_t P, int64_t stride_p, int64_t stride_t, int t0, int t1, int D) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) sum[i] = 0.f;
    for (int64_t t = (int64_t)t0 + (lane & 3); t < t1; t += 4) {
        const int64_t j = t / P;
        int64_t page = table[j];
        if (page < 0 || page >= num_slots) page = 0;
        const int64_t row = page * stride_p + (t - j * P) * stride_t + (lane >> 2);
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
            const float x = i * 8 < D ? load_elt(v, row + i * 8, kBf16 ? RKV_BF16 : RKV_F16) : 0.f;
            sum[i] += isfinite(x) ? 0.f : x;
        }
    }
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) {
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
    }
}

// kWhole: pages hold a multiple of 16 tokens, so 16 rows have one page (16 requests of up to 16384
// tokens, 16 heads on each of 2 x 128: 19.6 us, 20.1 with a page per row; long ones alike).
template <bool kBf16, int DP, int NH, int TT, int NW, int STAGES, bool kWhole>
__global__ void __launch_bounds__(NW * 32, 1)
decode_tc_kernel(DecodeParams p, int groups, Whole upto) {
    using Shape = TcShape<DP, NH, TT, NW, STAGES>;
    static_assert(TT % 16 == 0 && TT <= 32 && DP % 64 == 0 && (NH == 1 || NH == 2), "shape");
    extern __shared__ __align__(128) char smem[];
    __shared__ Left left[NW];
    constexpr int MH = NH * 8;
    constexpr int kChunks = DP / 8;             // 16-byte chunks per row
    constexpr int kCopies = 16 * kChunks / 32;  // copies per lane for 16 rows of K, and of V
    static_assert(STAGES * Shape::kStage / 2 >= Part::floats(MH, DP) * 4 && STAGES * Shape::kStage % 32 == 0,
                  "two parts fit the warp's ring");
    constexpr float kBias = tc_bias(kBf16);
    sm100::grid_launch_dependents();
    sm100::grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int G = p.Hq / p.Hkv;
    const Workspace ws(p, MH);

    const Runs runs = find_runs<TT, NW>(p, groups, upto);
    if (blockIdx.x >= runs.ctas) {
        if (threadIdx.x == 0) ws.open[blockIdx.x] = make_int4(-1, 0, 0, 0);
        return;
    }
    const uint32_t ring = sm100::smem_u32(smem) + warp * STAGES * Shape::kStage;
    const float scale2 = p.scale * kLog2e;
    const float slack = kSlack / scale2;
    Left mine{};
    // at the end of the run the ring is free and has room for two parts
    float* places = reinterpret_cast<float*>(smem + warp * STAGES * Shape::kStage);
    constexpr int kPlace = STAGES * Shape::kStage / 8;
    if (runs.count > 0) {
        const int count = (int)runs.count;
        Walk<TT> put, get;
        put.start(runs, groups);
        get = put;

        // ---- loads.  The lanes hold the ids of 32 pages in a row of the request, from page
        // `win_at` on; lane r looks up row r of the tile there (kWhole: row 16 r, for 16 rows).
        int ahead = count;
        const uint32_t P = (uint32_t)p.P;
        int64_t window = 0;
        uint32_t win_at = 0;
        int win_b = -1;
        const char* kbytes = static_cast<const char*>(p.k);
        const int64_t v_from_k = static_cast<const char*>(p.v) - kbytes;
        const int64_t row_bytes = p.stride_t * 2;
        constexpr int kStep = 32 / kChunks > 0 ? 32 / kChunks : 1;     // rows between a lane's copies
        const int lane_row = kChunks >= 32 ? 0 : lane / kChunks, lane_chunk = lane % kChunks;
        const uint32_t lane_dst = lane_row * Shape::kPitch + lane_chunk * 16;
        const int64_t lane_src = lane_row * row_bytes + lane_chunk * 16;
        const bool in_row = lane_chunk * 8 < p.D;
        // A segment's queries come with the first of its tiles in the run: a load of their own would
        // stand behind the copies that are under way.
        bool with_q = true;
        auto issue = [&](int stage) {
            if (ahead > 0) {
                const int t0 = put.token0();
                if (with_q) {
                    const int g0 = put.gi * MH, ng = min(MH, G - g0);
                    const char* src = static_cast<const char*>(p.q) +
                                      ((int64_t)put.b * p.q_stride_b + (int64_t)(put.h * G + g0) * p.q_stride_h) * 2;
                    const uint32_t to = ring + stage * Shape::kStage + 2 * Shape::kPlane;
#pragma unroll
                    for (int j = 0; j < MH * kChunks / 32; ++j) {
                        const int i = lane + 32 * j, r = i / kChunks, c = i % kChunks;
                        copy16_or_zero(to + r * Shape::kPitch + c * 16, src + r * p.q_stride_h * 2 + c * 16,
                                       r < ng && c * 8 < p.D);
                    }
                }
                const uint32_t p0 = p.div_p(max(t0, put.first));
                const uint32_t p1 = p.div_p(max(min(t0 + TT, put.last) - 1, 0));
                if (put.last > put.first && (put.b != win_b || p0 < win_at || p1 >= win_at + 32)) {
                    win_b = put.b;
                    win_at = p0;
                    const int64_t at = (int64_t)p0 + lane;
                    window = at * P < put.last ? p.table[(int64_t)put.b * p.table_stride + at] : 0;
                    if (window < 0 || window >= p.num_slots) { atomicMax(&g_error, kErrPage); window = 0; }
                }
                const int tr = t0 + (kWhole ? lane * 16 : lane);
                const uint32_t pr = p.div_p(tr);
                const int64_t page = __shfl_sync(0xffffffffu, window, pr - win_at);
                // byte offset of this lane's row (group of rows) in the pool
                const int64_t row = (page * p.stride_p + (int64_t)((uint32_t)tr - pr * P) * p.stride_t +
                                     (int64_t)put.h * p.stride_h) * 2;
                const uint32_t dst = ring + stage * Shape::kStage + lane_dst;
                // rows of the tile that this lane's copies read: [lo, lo + n), counted from its first
                const int lo = put.first - t0 - lane_row;
                const uint32_t n = in_row ? max(put.last - put.first, 0) : 0;
                if (kWhole) {
#pragma unroll
                    for (int x = 0; x < TT / 16; ++x) {
                        const char* src = kbytes + __shfl_sync(0xffffffffu, row, x) + lane_src;
                        const uint32_t to = dst + x * 16 * Shape::kPitch;
#pragma unroll
                        for (int j = 0; j < kCopies; ++j) {
                            const bool on = (uint32_t)(x * 16 + j * kStep - lo) < n;
                            copy16_or_zero(to + j * kStep * Shape::kPitch, src, on);
                            copy16_or_zero(to + Shape::kPlane + j * kStep * Shape::kPitch, src + v_from_k, on);
                            src += kStep * row_bytes;
                        }
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < kCopies * (TT / 16); ++j) {
                        const bool on = (uint32_t)(j * kStep - lo) < n;
                        const char* src = kbytes + __shfl_sync(0xffffffffu, row, lane_row + j * kStep) + lane_chunk * 16;
                        copy16_or_zero(dst + j * kStep * Shape::kPitch, src, on);
                        copy16_or_zero(dst + Shape::kPlane + j * kStep * Shape::kPitch, src + v_from_k, on);
                    }
                }
                --ahead;
                put.next(p, groups);
                with_q = put.tile == 0;
            }
            copies_commit();
        };

        // ---- products
        const int g = lane >> 2, c2 = (lane & 3) * 2;
        uint32_t q[DP / 16][NH][2];
#pragma unroll
        for (int s = 0; s < STAGES; ++s) issue(s);

        // column x of head block n: the logit (unscaled, as they all are) that is the base, and this
        // lane's share of the sum (zero: no logit seen)
        float o[DP / 16][NH][4], base[NH][2], l[NH][2];
        auto reset = [&]() {
#pragma unroll
            for (int n = 0; n < NH; ++n) {
#pragma unroll
                for (int d = 0; d < DP / 16; ++d)
#pragma unroll
                    for (int x = 0; x < 4; ++x) o[d][n][x] = 0.f;
#pragma unroll
                for (int x = 0; x < 2; ++x) { base[n][x] = -FLT_MAX; l[n][x] = 0.f; }
            }
        };
        reset();
        // ldmatrix rows of this lane: K (token, dim) as A, V (token, dim) transposed as A, and
        // queries (head, dim) as B
        const uint32_t q_lane = ring + 2 * Shape::kPlane + (lane & 7) * Shape::kPitch + (lane >> 3) * 16;
        const uint32_t k_lane = ring + (lane & 15) * Shape::kPitch + (lane >> 4) * 16;
        const uint32_t v_lane = ring + Shape::kPlane +
                                ((lane & 7) + (lane >> 4) * 8) * Shape::kPitch + ((lane >> 3) & 1) * 16;
        int tile_in = get.tile;     // the segment's first tile in this run
        int stage = 0;
        for (int i = 0; i < count; ++i) {
            copies_wait<STAGES - 1>();
            __syncwarp();
            if (get.tile == tile_in) {
#pragma unroll
                for (int n = 0; n < NH; ++n)
#pragma unroll
                    for (int k = 0; k < DP / 32; ++k)
                        sm100::ldsm_x4(q_lane + stage * Shape::kStage + n * 8 * Shape::kPitch + k * 64,
                                       q[2 * k][n][0], q[2 * k][n][1], q[2 * k + 1][n][0], q[2 * k + 1][n][1]);
            }
            const uint32_t kt = k_lane + stage * Shape::kStage, vt = v_lane + stage * Shape::kStage;
            float s[TT / 16][NH][4];
#pragma unroll
            for (int y = 0; y < TT / 16; ++y)
#pragma unroll
                for (int n = 0; n < NH; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x) s[y][n][x] = 0.f;
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
#pragma unroll
                for (int y = 0; y < TT / 16; ++y) {
                    uint32_t a0, a1, a2, a3;
                    sm100::ldsm_x4(kt + y * 16 * Shape::kPitch + k * 32, a0, a1, a2, a3);
#pragma unroll
                    for (int n = 0; n < NH; ++n)
                        sm100::mma_16816<kBf16>(s[y][n], a0, a1, a2, a3, q[k][n][0], q[k][n][1]);
                }
            }
            const int t0 = get.token0();
            if (t0 < get.first || t0 + TT > get.last) {
#pragma unroll
                for (int y = 0; y < TT / 16; ++y) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int t = t0 + y * 16 + g + (x / 2) * 8;
                        if (t < get.first || t >= get.last) {
#pragma unroll
                            for (int n = 0; n < NH; ++n) s[y][n][x] = -INFINITY;
                        }
                    }
                }
            }
            float top[NH][2];
            bool over = false;
#pragma unroll
            for (int n = 0; n < NH; ++n) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float v = fmaxf(s[0][n][x], s[0][n][x + 2]);
                    if constexpr (TT == 32) v = fmaxf(v, fmaxf(s[1][n][x], s[1][n][x + 2]));
                    top[n][x] = v;
                    over = over || v > base[n][x] + slack;
                }
            }
            if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                for (int n = 0; n < NH; ++n) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float v = top[n][x];
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
                        const bool renew = v > base[n][x] + slack;
                        const float alpha =
                            !renew ? 1.f : sm100::ex2((base[n][x] - v) * scale2);
                        base[n][x] = renew ? v : base[n][x];
                        l[n][x] *= alpha;
#pragma unroll
                        for (int d = 0; d < DP / 16; ++d) {
                            o[d][n][x] *= alpha;
                            o[d][n][x + 2] *= alpha;
                        }
                    }
                }
            }
#pragma unroll
            for (int y = 0; y < TT / 16; ++y) {
                uint32_t hi[NH][2], lo[NH][2];
#pragma unroll
                for (int n = 0; n < NH; ++n) {
#pragma unroll
                    for (int z = 0; z < 2; ++z) {   // tokens g, g + 8
                        const float w0 = sm100::ex2(fmaf(s[y][n][2 * z] - base[n][0], scale2, kBias));
                        const float w1 = sm100::ex2(fmaf(s[y][n][2 * z + 1] - base[n][1], scale2, kBias));
                        l[n][0] += w0;
                        l[n][1] += w1;
                        const uint32_t h = pack16<kBf16>(w0, w1);
                        const float2 back = unpack16<kBf16>(h);
                        hi[n][z] = sm100::movmatrix_trans(h);
                        lo[n][z] = sm100::movmatrix_trans(pack16<kBf16>(w0 - back.x, w1 - back.y));
                    }
                }
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) {
                    uint32_t a0, a1, a2, a3;
                    sm100::ldsm_x4_trans(vt + y * 16 * Shape::kPitch + d * 32, a0, a1, a2, a3);
#pragma unroll
                    for (int n = 0; n < NH; ++n) {
                        sm100::mma_16816<kBf16>(o[d][n], a0, a1, a2, a3, hi[n][0], hi[n][1]);
                        sm100::mma_16816<kBf16>(o[d][n], a0, a1, a2, a3, lo[n][0], lo[n][1]);
                    }
                }
            }
            __syncwarp();
            issue(stage);
            stage = stage + 1 == STAGES ? 0 : stage + 1;

            // ---- the end of the segment, or of the run
            const bool ends = get.tile + 1 == get.tiles, last = i + 1 == count;
            if (ends || last) {
                const bool whole = tile_in == 0 && ends;
                const int h = get.h, g0 = get.gi * MH;
                const int ng = min(MH, G - g0);
                if (!whole) {
                    if (tile_in > 0) {
                        mine.head = 1; mine.ends = ends; mine.early = !last;
                        mine.head_b = get.b; mine.head_seg = h * groups + get.gi;
                    } else {
                        mine.tail = 1; mine.tail_b = get.b; mine.tail_seg = h * groups + get.gi;
                    }
                    mine.rest = get.tiles - get.tile - 1;
                }
                const Part part = last ? Part{places, MH, p.D}
                                       : ws.warp((int64_t)blockIdx.x * NW + warp);
                float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int n = 0; n < NH; ++n) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        l[n][x] += __shfl_xor_sync(0xffffffffu, l[n][x], 4);
                        l[n][x] += __shfl_xor_sync(0xffffffffu, l[n][x], 8);
                        l[n][x] += __shfl_xor_sync(0xffffffffu, l[n][x], 16);
                    }
#pragma unroll
                    for (int d = 0; d < DP / 16; ++d)
#pragma unroll
                        for (int x = 0; x < 4; ++x) zero[x] = fmaf(o[d][n][x], 0.f, zero[x]);
                }
                bool odd = false;       // an infinity or NaN, and weights that are none
#pragma unroll
                for (int n = 0; n < NH; ++n) odd = odd || l[n][0] > 0.f || l[n][1] > 0.f;
                odd = odd && (zero[0] + zero[1]) + (zero[2] + zero[3]) != 0.f;
                if (__any_sync(0xffffffffu, odd)) {
                    float sum[DP / 8];
                    const int from = max(get.first, (int)(((uint32_t)get.first / TT + tile_in) * TT));
                    odd_columns<kBf16, DP>(sum, static_cast<const char*>(p.v) + (int64_t)h * p.stride_h * 2,
                                           p.table + (int64_t)get.b * p.table_stride, p.num_slots, p.P, p.stride_p,
                                           p.stride_t, from, min(get.last, t0 + TT), p.D);
#pragma unroll
                    for (int n = 0; n < NH; ++n)
#pragma unroll
                        for (int d = 0; d < DP / 16; ++d)
#pragma unroll
                            for (int x = 0; x < 4; ++x)
                                if (l[n][x & 1] > 0.f && isnan(o[d][n][x]) && sum[2 * d + x / 2] != 0.f)
                                    o[d][n][x] = sum[2 * d + x / 2];
                }
#pragma unroll
                for (int n = 0; n < NH; ++n) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float sum = l[n][x];
                        const int row = 8 * n + c2 + x;
                        const float b = l[n][x] == 0.f ? -INFINITY : base[n][x];
                        if (g == 0 && row < ng) {
                            if (!whole) { part.top(row) = b; part.sum(row) = sum; }
                            else if (p.lse) p.lse[(int64_t)get.b * p.Hq + h * G + g0 + row] = lse_of(p, b, sum);
                        }
                        if (whole) {
                            const float inv = sum == 0.f ? 0.f : __frcp_rn(sum);
#pragma unroll
                            for (int d = 0; d < DP / 16; ++d) {
                                o[d][n][x] *= inv;
                                o[d][n][x + 2] *= inv;
                            }
                        } else if (row < ng) {
                            float* acc = part.acc(row) + g;
#pragma unroll
                            for (int d = 0; d < DP / 16; ++d) {
                                if (d * 16 < p.D) acc[d * 16] = o[d][n][x];
                                if (d * 16 + 8 < p.D) acc[d * 16 + 8] = o[d][n][x + 2];
                            }
                        }
                    }
                    if (whole) {
                        // dims in pairs, heads over the lanes
                        const int row = 8 * n + g;
                        char* out = static_cast<char*>(p.out) +
                                    ((int64_t)get.b * p.o_stride_b +
                                     (int64_t)(h * G + g0 + row) * p.o_stride_h + c2) * 2;
#pragma unroll
                        for (int d = 0; d < DP / 16; ++d) {
#pragma unroll
                            for (int z = 0; z < 2; ++z) {
                                const uint32_t v = sm100::movmatrix_trans(
                                    pack16<kBf16>(o[d][n][2 * z], o[d][n][2 * z + 1]));
                                if (row < ng && d * 16 + z * 8 < p.D)
                                    *reinterpret_cast<uint32_t*>(out + (d * 16 + z * 8) * 2) = v;
                            }
                        }
                    }
                }
                reset();
                tile_in = 0;
            }
            get.next(p, groups);
        }
    }
    if (mine.early) {   // a head that ended while the ring was in use comes back
        __syncwarp();
        const float4* from = reinterpret_cast<const float4*>(ws.warp((int64_t)blockIdx.x * NW + warp).at);
        for (int i = lane; i < Part::floats(MH, p.D) / 4; i += 32)
            reinterpret_cast<float4*>(places + kPlace)[i] = from[i];
    }
    if (lane == 0) left[warp] = mine;
    __syncthreads();
    join_parts<NW, MH, kBf16 ? RKV_BF16 : RKV_F16>(p, runs, ws, left, reinterpret_cast<float*>(smem),
                                                   2 * kPlace, kPlace, groups);
}

// ------------------------------------------------------------------------------------------
// fp32.  The same rings, with fp32 arithmetic (a product of tensor cores would round K and V to
// fewer bits).  For the logits, LPT lanes share a token and read its row a quarter (half) each,
// the queries come as broadcasts; for the output, a lane has DP / 32 dims of every head.  Both
// halves are fused multiply-adds on pairs.  Up to 4 heads per kv head memory is the bound (8
// requests of 9155 tokens, 4 kv heads x 128: 54 us, 5.6 TB/s), with 8 the instructions are (72 us).
// ------------------------------------------------------------------------------------------
template <int DP, int HG, int TT, int NW, int STAGES>
struct F32Shape {
    static constexpr int kLpt = 32 / TT;                // lanes per token
    static constexpr int kPitch = DP * 4 + 16 * kLpt;   // 8 lanes at a time read 128 different bytes
    static constexpr int kPlane = TT * kPitch;
    // Queries come with the first tile of their segment; with 8 heads of 256 dims there is no room for
    // them, and 8 heads read them when the segment begins (8 requests of 9155 tokens, 4 kv heads x 128:
    // 72.2 us, where they would fit, and take 69.3, with the tile).
    static constexpr bool kQInRing = HG <= 4;
    static constexpr int kStage = 2 * kPlane + (kQInRing ? HG * kPitch : 0);
    static constexpr int kSmem = NW * (STAGES * kStage + HG * kPitch);
};

template <int DP, int HG, int TT, int NW, int STAGES>
__global__ void __launch_bounds__(NW * 32, 1)
decode_f32_kernel(DecodeParams p, int groups, Whole upto) {
    using Shape = F32Shape<DP, HG, TT, NW, STAGES>;
    static_assert(HG % 4 == 0 && DP % 64 == 0 && (TT == 8 || TT == 16), "shape");
    extern __shared__ __align__(128) char smem[];
    __shared__ Left left[NW];
    __shared__ __align__(16) float s_weight[NW][TT][HG];
    constexpr int kLpt = Shape::kLpt;
    constexpr int kChunks = DP / 4;                 // 16-byte chunks per row
    constexpr int kCopies = TT * kChunks / 32;      // copies per lane for K, and for V
    constexpr int kDims = DP / 32;                  // dims per lane of the output
    constexpr int kPlace = STAGES * Shape::kStage / 8;
    static_assert(kPlace >= Part::floats(HG, DP) && STAGES * Shape::kStage % 32 == 0, "two parts fit the ring");
    sm100::grid_launch_dependents();
    sm100::grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int G = p.Hq / p.Hkv;
    const Workspace ws(p, HG);
    const Runs runs = find_runs<TT, NW>(p, groups, upto);
    if (blockIdx.x >= runs.ctas) {
        if (threadIdx.x == 0) ws.open[blockIdx.x] = make_int4(-1, 0, 0, 0);
        return;
    }
    const uint32_t ring = sm100::smem_u32(smem) + warp * STAGES * Shape::kStage;
    float* places = reinterpret_cast<float*>(smem + warp * STAGES * Shape::kStage);
    const float scale2 = p.scale * kLog2e, slack = kSlack / scale2;
    Left mine{};
    if (runs.count > 0) {
        const int count = (int)runs.count;
        Walk<TT> put, get;
        put.start(runs, groups);
        get = put;
        int ahead = count;
        const uint32_t P = (uint32_t)p.P;
        int64_t window = 0;     // ids of 32 pages in a row, from page `win_at` of request win_b on
        uint32_t win_at = 0;
        int win_b = -1;
        const char* kbytes = static_cast<const char*>(p.k);
        const int64_t v_from_k = static_cast<const char*>(p.v) - kbytes;
        bool with_q = true;     // queries come with the first tile of their segment
        auto issue = [&](int stage) {
            if (ahead > 0) {
                const int t0 = put.token0();
                const uint32_t dst = ring + stage * Shape::kStage;
                if (Shape::kQInRing && with_q) {
                    const int g0 = put.gi * HG, ng = min(HG, G - g0);
                    const char* src = static_cast<const char*>(p.q) +
                                      ((int64_t)put.b * p.q_stride_b + (int64_t)(put.h * G + g0) * p.q_stride_h) * 4;
#pragma unroll
                    for (int j = 0; j < HG * kChunks / 32; ++j) {
                        const int i = lane + 32 * j, r = i / kChunks, c = i % kChunks;
                        copy16_or_zero(dst + 2 * Shape::kPlane + r * Shape::kPitch + c * 16,
                                       src + r * p.q_stride_h * 4 + c * 16, r < ng && c * 4 < p.D);
                    }
                }
                const uint32_t p0 = p.div_p(max(t0, put.first));
                const uint32_t p1 = p.div_p(max(min(t0 + TT, put.last) - 1, 0));
                if (put.last > put.first && (put.b != win_b || p0 < win_at || p1 >= win_at + 32)) {
                    win_b = put.b;
                    win_at = p0;
                    const int64_t at = (int64_t)p0 + lane;
                    window = at * P < put.last ? p.table[(int64_t)put.b * p.table_stride + at] : 0;
                    if (window < 0 || window >= p.num_slots) { atomicMax(&g_error, kErrPage); window = 0; }
                }
                // byte offset of row `lane` of the tile in the pool
                const int tr = t0 + lane;
                const uint32_t pr = p.div_p(tr);
                const int64_t page = __shfl_sync(0xffffffffu, window, pr - win_at);
                const int64_t row = (page * p.stride_p + (int64_t)((uint32_t)tr - pr * P) * p.stride_t +
                                     (int64_t)put.h * p.stride_h) * 4;
#pragma unroll
                for (int j = 0; j < kCopies; ++j) {
                    const int i = lane + 32 * j, r = i / kChunks, c = i % kChunks;
                    const bool on = t0 + r >= put.first && t0 + r < put.last && c * 4 < p.D;
                    const char* src = kbytes + __shfl_sync(0xffffffffu, row, r) + c * 16;
                    copy16_or_zero(dst + r * Shape::kPitch + c * 16, src, on);
                    copy16_or_zero(dst + Shape::kPlane + r * Shape::kPitch + c * 16, src + v_from_k, on);
                }
                --ahead;
                put.next(p, groups);
                with_q = put.tile == 0;
            }
            copies_commit();
        };
#pragma unroll
        for (int s = 0; s < STAGES; ++s) issue(s);

        const int tok = lane / kLpt, share = lane % kLpt;
        uint64_t o[HG][kDims / 2];
        float base[HG], limit[HG], l[HG];
        auto reset = [&]() {
#pragma unroll
            for (int g = 0; g < HG; ++g) {
                base[g] = 0.f; limit[g] = -INFINITY; l[g] = 0.f;
#pragma unroll
                for (int x = 0; x < kDims / 2; ++x) o[g][x] = 0;
            }
        };
        reset();
        const uint32_t k_lane = ring + tok * Shape::kPitch + share * 16;
        // dims of this lane: two, or fours that are 128 apart
        const uint32_t v_lane = ring + Shape::kPlane + lane * (kDims == 2 ? 8 : 16);
        int tile_in = get.tile, stage = 0;
        // the queries are moved from the stage that brought them to a place behind the rings
        float* q_own = reinterpret_cast<float*>(smem + NW * STAGES * Shape::kStage) + warp * HG * (Shape::kPitch / 4);
        const uint32_t q_base = sm100::smem_u32(q_own) + share * 16;
        for (int i = 0; i < count; ++i) {
            copies_wait<STAGES - 1>();
            __syncwarp();
            const uint32_t at = stage * Shape::kStage;
            if (get.tile == tile_in) {
                if constexpr (Shape::kQInRing) {
                    for (int x = lane; x < HG * Shape::kPitch / 16; x += 32)
                        reinterpret_cast<uint4*>(q_own)[x] = sm100::lds128(ring + at + 2 * Shape::kPlane + x * 16);
                } else {
                    const int g0 = get.gi * HG, ng = min(HG, G - g0);
                    const float* src = static_cast<const float*>(p.q) + (int64_t)get.b * p.q_stride_b +
                                       (int64_t)(get.h * G + g0) * p.q_stride_h;
#pragma unroll
                    for (int j = 0; j < HG * kChunks / 32; ++j) {
                        const int x = lane + 32 * j, r = x / kChunks, c = x % kChunks;
                        const float4 v = r < ng && c * 4 < p.D
                                             ? *reinterpret_cast<const float4*>(src + r * p.q_stride_h + c * 4)
                                             : make_float4(0.f, 0.f, 0.f, 0.f);
                        *reinterpret_cast<float4*>(q_own + r * (Shape::kPitch / 4) + c * 4) = v;
                    }
                }
                __syncwarp();
            }
            uint64_t s2[HG];
#pragma unroll
            for (int g = 0; g < HG; ++g) s2[g] = 0;
#pragma unroll
            for (int j = 0; j < kChunks / kLpt; ++j) {
                const uint4 k = sm100::lds128(k_lane + at + j * kLpt * 16);
                const uint64_t k0 = (uint64_t)k.y << 32 | k.x, k1 = (uint64_t)k.w << 32 | k.z;
#pragma unroll
                for (int g = 0; g < HG; ++g) {
                    const uint4 q = sm100::lds128(q_base + g * Shape::kPitch + j * kLpt * 16);
                    sm100::ffma2(s2[g], (uint64_t)q.y << 32 | q.x, k0);
                    sm100::ffma2(s2[g], (uint64_t)q.w << 32 | q.z, k1);
                }
            }
            const int t = get.token0() + tok;
            const bool in = t >= get.first && t < get.last;
            float s[HG];
            bool over = false;
#pragma unroll
            for (int g = 0; g < HG; ++g) {
                float v = sm100::sum_pair(s2[g]);
#pragma unroll
                for (int x = kLpt / 2; x > 0; x >>= 1) v += __shfl_xor_sync(0xffffffffu, v, x);
                s[g] = in ? v : -INFINITY;
                over = over || s[g] > limit[g];
            }
            if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                for (int g = 0; g < HG; ++g) {
                    float v = s[g];
#pragma unroll
                    for (int x = 16; x >= kLpt; x >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, x));
                    const bool renew = v > limit[g];
                    const float alpha = !renew ? 1.f : limit[g] == -INFINITY ? 0.f : sm100::ex2((base[g] - v) * scale2);
                    base[g] = renew ? v : base[g];
                    limit[g] = renew ? v + slack : limit[g];
                    l[g] *= alpha;
#pragma unroll
                    for (int x = 0; x < kDims / 2; ++x) o[g][x] = sm100::fmul2(o[g][x], sm100::pack2(alpha, alpha));
                }
            }
#pragma unroll
            for (int g = 0; g < HG; ++g) {
                s[g] = sm100::ex2((s[g] - base[g]) * scale2);
                l[g] += s[g];
            }
            if (share == 0) {
#pragma unroll
                for (int g = 0; g < HG; g += 4)
                    *reinterpret_cast<float4*>(&s_weight[warp][tok][g]) = make_float4(s[g], s[g + 1], s[g + 2], s[g + 3]);
            }
            __syncwarp();
#pragma unroll
            for (int y = 0; y < TT; ++y) {
                uint64_t v[kDims / 2];
                if constexpr (kDims == 2) {
                    v[0] = (uint64_t)sm100::lds32(v_lane + at + y * Shape::kPitch + 4) << 32 |
                           sm100::lds32(v_lane + at + y * Shape::kPitch);
                } else {
#pragma unroll
                    for (int x = 0; x < kDims / 4; ++x) {
                        const uint4 f = sm100::lds128(v_lane + at + y * Shape::kPitch + x * 512);
                        v[2 * x] = (uint64_t)f.y << 32 | f.x;
                        v[2 * x + 1] = (uint64_t)f.w << 32 | f.z;
                    }
                }
#pragma unroll
                for (int g = 0; g < HG; g += 4) {
                    const float4 w = *reinterpret_cast<const float4*>(&s_weight[warp][y][g]);
#pragma unroll
                    for (int x = 0; x < kDims / 2; ++x) {
                        sm100::ffma2(o[g][x], sm100::pack2(w.x, w.x), v[x]);
                        sm100::ffma2(o[g + 1][x], sm100::pack2(w.y, w.y), v[x]);
                        sm100::ffma2(o[g + 2][x], sm100::pack2(w.z, w.z), v[x]);
                        sm100::ffma2(o[g + 3][x], sm100::pack2(w.w, w.w), v[x]);
                    }
                }
            }
            __syncwarp();
            issue(stage);
            stage = stage + 1 == STAGES ? 0 : stage + 1;

            // ---- the end of the segment, or of the run
            const bool ends = get.tile + 1 == get.tiles, last = i + 1 == count;
            if (ends || last) {
                const bool whole = tile_in == 0 && ends;
                const int h = get.h, g0 = get.gi * HG;
                const int ng = min(HG, G - g0);
                if (!whole) {
                    if (tile_in > 0) {
                        mine.head = 1; mine.ends = ends; mine.early = !last;
                        mine.head_b = get.b; mine.head_seg = h * groups + get.gi;
                    } else {
                        mine.tail = 1; mine.tail_b = get.b; mine.tail_seg = h * groups + get.gi;
                    }
                    mine.rest = get.tiles - get.tile - 1;
                }
                const Part part = last ? Part{places, HG, p.D} : ws.warp((int64_t)blockIdx.x * NW + warp);
#pragma unroll
                for (int g = 0; g < HG; ++g) {
                    float sum = l[g];
#pragma unroll
                    for (int x = 16; x >= kLpt; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
                    if (g >= ng) break;
                    const int hq = h * G + g0 + g;
                    const float b = limit[g] == -INFINITY ? -INFINITY : base[g];
                    if (lane == 0) {
                        if (!whole) { part.top(g) = b; part.sum(g) = sum; }
                        else if (p.lse) p.lse[(int64_t)get.b * p.Hq + hq] = lse_of(p, b, sum);
                    }
                    const float inv = !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
                    float* to = whole ? static_cast<float*>(p.out) + (int64_t)get.b * p.o_stride_b + (int64_t)hq * p.o_stride_h
                                      : part.acc(g);
#pragma unroll
                    for (int x = 0; x < kDims / 2; ++x) {
                        const int d = kDims == 2 ? lane * 2 : (x / 2) * 128 + lane * 4 + (x % 2) * 2;
                        const uint64_t v = sm100::fmul2(o[g][x], sm100::pack2(inv, inv));
                        if (d < p.D) *reinterpret_cast<uint64_t*>(to + d) = v;
                    }
                }
                reset();
                tile_in = 0;
            }
            get.next(p, groups);
        }
    }
    if (mine.early) {   // a head that ended while the ring was in use comes back
        __syncwarp();
        const float4* from = reinterpret_cast<const float4*>(ws.warp((int64_t)blockIdx.x * NW + warp).at);
        for (int i = lane; i < Part::floats(HG, p.D) / 4; i += 32)
            reinterpret_cast<float4*>(places + kPlace)[i] = from[i];
    }
    if (lane == 0) left[warp] = mine;
    __syncthreads();
    join_parts<NW, HG, RKV_F32>(p, runs, ws, left, reinterpret_cast<float*>(smem), 2 * kPlace, kPlace, groups);
}

// ------------------------------------------------------------------------------------------
// Every other shape: any alignment, head_dim up to 256.  Lanes share the elements of a row; a
// token's logit is a sum over the warp.
// ------------------------------------------------------------------------------------------
constexpr int kAnyTile = 16, kAnyWarps = 8, kAnyHeads = 4;

__global__ void __launch_bounds__(kAnyWarps * 32)
decode_any_kernel(DecodeParams p, int groups, Whole upto) {
    constexpr int HG = kAnyHeads, kPlace = Part::floats(HG, kMaxHeadDim);
    extern __shared__ __align__(128) char smem[];
    __shared__ Left left[kAnyWarps];
    sm100::grid_launch_dependents();
    sm100::grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Workspace ws(p, HG);
    const Runs runs = find_runs<kAnyTile, kAnyWarps>(p, groups, upto);
    if (blockIdx.x >= runs.ctas) {
        if (threadIdx.x == 0) ws.open[blockIdx.x] = make_int4(-1, 0, 0, 0);
        return;
    }
    const int G = p.Hq / p.Hkv;
    const int ne = (p.D + 31) / 32;
    const float scale2 = p.scale * kLog2e;
    float* places = reinterpret_cast<float*>(smem) + warp * 2 * kPlace;
    Left mine{};
    int b = runs.b, h = runs.seg / groups, gi = runs.seg % groups;
    int64_t tile0 = runs.tile, tiles = runs.tiles, first = runs.first, last = runs.last;
    for (int64_t todo = runs.count; todo > 0;) {
        const int64_t tile1 = min(tiles, tile0 + todo);
        const int64_t* table = p.table + (int64_t)b * p.table_stride;
        const int g0 = gi * HG, ng = min(HG, G - g0);
        const int64_t q0 = (int64_t)b * p.q_stride_b + (int64_t)(h * G + g0) * p.q_stride_h;
        float q[HG][8], acc[HG][8], m[HG], l[HG];
#pragma unroll
        for (int g = 0; g < HG; ++g) {
            m[g] = -INFINITY;
            l[g] = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = lane + 32 * i;
                q[g][i] = g < ng && e < p.D ? load_elt(p.q, q0 + g * p.q_stride_h + e, p.dtype) : 0.f;
                acc[g][i] = 0.f;
            }
        }
        const int64_t t1 = min(last, (first / kAnyTile + tile1) * kAnyTile);
        for (int64_t t = max(first, (first / kAnyTile + tile0) * kAnyTile); t < t1; ++t) {
            const int64_t j = t / p.P;
            int64_t page = table[j];
            if (page < 0 || page >= p.num_slots) { atomicMax(&g_error, kErrPage); page = 0; }
            const int64_t off = page * p.stride_p + (t - j * p.P) * p.stride_t + (int64_t)h * p.stride_h;
            float kr[8], vr[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = lane + 32 * i;
                kr[i] = i < ne && e < p.D ? load_elt(p.k, off + e, p.dtype) : 0.f;
                vr[i] = i < ne && e < p.D ? load_elt(p.v, off + e, p.dtype) : 0.f;
            }
#pragma unroll
            for (int g = 0; g < HG; ++g) {
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) s = fmaf(q[g][i], kr[i], s);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
                const float mn = fmaxf(m[g], s);
                const float base = mn == -INFINITY ? 0.f : mn;
                const float alpha = sm100::ex2((m[g] - base) * scale2), w = sm100::ex2((s - base) * scale2);
                m[g] = mn;
                l[g] = l[g] * alpha + w;
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[g][i] = acc[g][i] * alpha + w * vr[i];
            }
        }
        todo -= tile1 - tile0;
        const bool ends = tile1 == tiles, whole = tile0 == 0 && ends;
        const bool is_early = !whole && tile0 > 0 && todo > 0;
        if (!whole) {
            if (tile0 > 0) {
                mine.head = 1; mine.ends = ends; mine.early = is_early;
                mine.head_b = b; mine.head_seg = h * groups + gi;
            } else {
                mine.tail = 1; mine.tail_b = b; mine.tail_seg = h * groups + gi;
            }
            mine.rest = tiles - tile1;
        }
        const Part part{places + (is_early ? kPlace : 0), HG, p.D};
#pragma unroll
        for (int g = 0; g < HG; ++g) {
            if (g >= ng) break;
            const int hq = h * G + g0 + g;
            const float inv = l[g] == 0.f ? 0.f : 1.f / l[g];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = lane + 32 * i;
                if (e >= p.D) break;
                if (whole)
                    store_elt(p.out, (int64_t)b * p.o_stride_b + (int64_t)hq * p.o_stride_h + e,
                              p.dtype, acc[g][i] * inv);
                else part.acc(g)[e] = acc[g][i];
            }
            if (lane == 0) {
                if (!whole) { part.top(g) = m[g]; part.sum(g) = l[g]; }
                else if (p.lse) p.lse[(int64_t)b * p.Hq + hq] = lse_of(p, m[g], l[g]);
            }
        }
        tile0 = 0;
        if (++gi == groups) {
            gi = 0;
            if (++h == p.Hkv) {
                h = 0;
                if (++b < p.B) {
                    range_of(p, b, &first, &last);
                    tiles = tiles_of<kAnyTile>(first, last);
                }
            }
        }
    }
    if (lane == 0) left[warp] = mine;
    __syncthreads();
    join_parts<kAnyWarps, HG, -1>(p, runs, ws, left, reinterpret_cast<float*>(smem), 2 * kPlace, kPlace, groups);
}

// ------------------------------------------------------------------------------------------
// CTA (c, row): row `row` of the segment that goes on behind the run of decode CTA c, if one
// does: its part there and one part of each CTA behind, at most kCtas in all.  The threads weigh
// the parts, and warp w sums the parts w, w + kMergeWarps, ..., whose sums are added in order.
// All of it is waiting for memory, so the first kMergeAhead parts of each warp are on their way
// before the weights are known.
// ------------------------------------------------------------------------------------------
constexpr int kMergeWarps = 4, kMergeAhead = 10, kMergeThreads = kMergeWarps * 32;
static_assert(2 * kMergeThreads >= kCtas, "a thread weighs up to two parts");

__global__ void __launch_bounds__(kMergeWarps * 32)
merge_kernel(DecodeParams p, int groups, int HG) {
    __shared__ float s_weight[2 * kMergeThreads], s_top[kMergeWarps], s_sum[kMergeWarps];
    __shared__ float s_acc[kMergeWarps][kMaxHeadDim];
    sm100::grid_launch_dependents();
    sm100::grid_dependency_wait();
    const Workspace ws(p, HG);
    const int c = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
    const int4 open = ws.open[c];
    if (open.x < 0) return;
    const int G = p.Hq / p.Hkv;
    const int h = groups == 1 ? open.y : open.y / groups, g0 = (open.y - h * groups) * HG, n = open.z + 1;
    if (g0 + row >= G) return;
    const int lane = tid & 31, warp = tid >> 5;
    // part 0 is the open one of CTA c, part i > 0 the first of CTA c + i
    const float* parts = ws.cta(c, 0).at;
    auto at = [&](int i) { return parts + (2 * i + (i == 0)) * ws.stride; };
    float2 ml[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int i = tid + k * kMergeThreads;
        ml[k] = i < n ? *reinterpret_cast<const float2*>(at(i) + 2 * row) : make_float2(-INFINITY, 0.f);
    }
    const int skip = 2 * HG + row * (p.D + 4) + lane;
    float ahead[kMergeAhead][4];
#pragma unroll
    for (int k = 0; k < kMergeAhead; ++k) {
        const float* f = at(min(warp + k * kMergeWarps, n - 1)) + skip;
#pragma unroll
        for (int x = 0; x < 4; ++x) ahead[k][x] = lane + 32 * x < p.D ? f[32 * x] : 0.f;
    }
    float top = fmaxf(ml[0].x, ml[1].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) s_top[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kMergeWarps; ++w) top = fmaxf(top, s_top[w]);
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float weight = part_weight(p, ml[k].x, top);
        s_weight[tid + k * kMergeThreads] = weight;
        if (tid + k * kMergeThreads < n) sum += ml[k].y * weight;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < kMergeWarps; ++w) sum += s_sum[w];
    for (int x0 = 0; x0 * 32 < p.D; x0 += 4) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        int i = warp;
        if (x0 == 0) {
#pragma unroll
            for (int k = 0; k < kMergeAhead; ++k, i += kMergeWarps)
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    if (i < n) acc[x] = fmaf(ahead[k][x], s_weight[i], acc[x]);
        }
#pragma unroll 4
        for (; i < n; i += kMergeWarps) {
            const float* f = at(i) + skip + 32 * x0;
            const float a = s_weight[i];
#pragma unroll
            for (int x = 0; x < 4; ++x)
                if (lane + 32 * (x0 + x) < p.D) acc[x] = fmaf(f[32 * x], a, acc[x]);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) s_acc[warp][lane + 32 * (x0 + x)] = acc[x];
    }
    __syncthreads();
    const int hq = h * G + g0 + row;
    for (int d = tid; d < p.D; d += kMergeThreads) {
        float o = 0.f;
#pragma unroll
        for (int w = 0; w < kMergeWarps; ++w) o += s_acc[w][d];
        store_elt(p.out, (int64_t)open.x * p.o_stride_b + (int64_t)hq * p.o_stride_h + d, p.dtype,
                  sum == 0.f ? 0.f : o / sum);
    }
    if (p.lse && tid == 0) p.lse[(int64_t)open.x * p.Hq + hq] = lse_of(p, top, sum);
}

namespace {

// 16-byte rows in the pool and in q (copies), 4-byte ones in out, token counts of 31 bits
bool tc_ok(const DecodeParams& p) {
    if (p.dtype == RKV_F32 || p.D % 8) return false;
    if (p.W * p.P > 0x7fffff00 || p.P > 0x7fffffff) return false;
    for (int64_t s : {p.stride_h, p.stride_p, p.stride_t, p.q_stride_b, p.q_stride_h})
        if (s % 8) return false;
    for (const void* ptr : {p.k, p.v, p.q})
        if (reinterpret_cast<uintptr_t>(ptr) & 15) return false;
    return p.o_stride_b % 2 == 0 && p.o_stride_h % 2 == 0 && !(reinterpret_cast<uintptr_t>(p.out) & 3);
}

// A decode kernel and its merge (where there can be something to join), each launched so that its start overlaps the end of the kernel
// before it (both wait for that kernel's results first).
template <void (*kernel)(DecodeParams, int, Whole)>
cudaError_t launch_pair(int threads, int smem, const DecodeParams& p, int HG, int TT, float bias, cudaStream_t st) {
    const int groups = (p.Hq / p.Hkv + HG - 1) / HG;
    // the kernel's shared memory is set once per device (a setting of the function, not of a call)
    static std::atomic<uint64_t> set{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !(set.load(std::memory_order_acquire) >> dev & 1)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        if (dev < 64) set.fetch_or(1ull << dev, std::memory_order_release);
    }
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(kCtas);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    DecodeParams q = p;
    q.bias = bias;
    // (units beyond the tiles of the table's capacity: one for a range that starts within a tile, one
    // or two for the segment itself; doubled, for the search that moves boundaries)
    q.narrow = (double)p.B * p.Hkv * groups * ((double)p.W * p.P / TT + 4) * 2 < 2147483647.0;
    // (a range of tokens that does not start at a tile's first reaches into one tile more)
    const int64_t most = (p.W * p.P + TT - 1) / TT + (p.starts ? 1 : 0);
    const Whole upto = whole_tiles((int64_t)p.B * p.Hkv * groups, most, threads / 32);
    e = counted(cudaLaunchKernelEx(&cfg, kernel, q, groups, upto), 1);
    if (e != cudaSuccess || most <= upto.cta) return e;
    cfg.gridDim = dim3(kCtas, HG);
    cfg.blockDim = dim3(kMergeWarps * 32);
    cfg.dynamicSmemBytes = 0;
    return counted(cudaLaunchKernelEx(&cfg, merge_kernel, q, groups, HG), 1);
}

template <bool kBf16, int DP, int NH, bool kWhole>
cudaError_t launch_tc(const DecodeParams& p, cudaStream_t st) {
    // Tiles of 16 KB of K and V a warp and two of them in its ring: 128 KB on their way per SM, where
    // 64 KB do not fill the memory (8 requests of 32768 tokens, 8 x 128: 181 us, and 208 with tiles of 16
    // tokens).  Four warps leave fewer parts to join than eight with tiles of 16 (1 request of 131072
    // tokens, 4 x 128: 53 and 56 us; 64 of 250, 8 x 128: 15.7 and 19.1), but 16 heads at a time are more
    // work per tile than one warp per scheduler does in time (64 requests of 500 tokens, 2 x 128: 23.9
    // and 21.2).
    constexpr bool kWide = DP == 128 && NH == 2;
    constexpr int TT = DP <= 128 && !kWide ? 32 : 16, NW = DP <= 64 || kWide ? 8 : 4, STAGES = 2;
    using Shape = TcShape<DP, NH, TT, NW, STAGES>;
    static_assert(NW <= kMostWarps && Shape::kSmem <= 232448 - 4096, "shared memory");
    return launch_pair<decode_tc_kernel<kBf16, DP, NH, TT, NW, STAGES, kWhole>>(NW * 32, Shape::kSmem, p, NH * 8, TT, tc_bias(kBf16), st);
}

template <int DP, int NH>
cudaError_t launch_tc_dim(const DecodeParams& p, cudaStream_t st) {
    const bool whole = p.P % 16 == 0;
    if (p.dtype == RKV_BF16) return whole ? launch_tc<true, DP, NH, true>(p, st) : launch_tc<true, DP, NH, false>(p, st);
    return whole ? launch_tc<false, DP, NH, true>(p, st) : launch_tc<false, DP, NH, false>(p, st);
}

template <int DP>
cudaError_t launch_tc_heads(const DecodeParams& p, cudaStream_t st) {
    return p.Hq / p.Hkv > 8 ? launch_tc_dim<DP, 2>(p, st) : launch_tc_dim<DP, 1>(p, st);
}

// The same for fp32, with rows of 16 bytes in out
bool f32_ok(const DecodeParams& p) {
    if (p.dtype != RKV_F32 || p.D % 4) return false;
    if (p.W * p.P > 0x7fffff00 || p.P > 0x7fffffff) return false;
    for (int64_t s : {p.stride_h, p.stride_p, p.stride_t, p.q_stride_b, p.q_stride_h, p.o_stride_b, p.o_stride_h})
        if (s % 4) return false;
    for (const void* ptr : {p.k, p.v, p.q, (const void*)p.out})
        if (reinterpret_cast<uintptr_t>(ptr) & 15) return false;
    return true;
}

template <int DP, int HG>
cudaError_t launch_f32(const DecodeParams& p, cudaStream_t st) {
    // (8 heads x 128: 72 us with four warps and tiles of 16 tokens, 76 with eight and 8)
    constexpr bool kWide = DP == 128 && HG == 8;
    constexpr int TT = DP <= 64 || kWide ? 16 : 8, NW = DP <= 128 && !kWide ? 8 : 4, STAGES = 2;
    using Shape = F32Shape<DP, HG, TT, NW, STAGES>;
    static_assert(NW <= kMostWarps && Shape::kSmem <= 232448 - 8192, "shared memory");
    return launch_pair<decode_f32_kernel<DP, HG, TT, NW, STAGES>>(NW * 32, Shape::kSmem, p, HG, TT, 0.f, st);
}

template <int DP>
cudaError_t launch_f32_heads(const DecodeParams& p, cudaStream_t st) {
    return p.Hq / p.Hkv > 4 ? launch_f32<DP, 8>(p, st) : launch_f32<DP, 4>(p, st);
}

}  // namespace

// Upper bound over the kernels that a call of these sizes may take.
size_t decode_workspace_bytes(int64_t Hq, int64_t Hkv, int64_t D) {
    return Workspace::bytes(kMostWarps, Hq / Hkv > 8 ? 16 : 8, D);
}

cudaError_t launch_decode(const DecodeParams& p, cudaStream_t st) {
    if (f32_ok(p)) {
        if (p.D <= 64) return launch_f32_heads<64>(p, st);
        if (p.D <= 128) return launch_f32_heads<128>(p, st);
        return launch_f32_heads<256>(p, st);
    }
    if (!tc_ok(p)) return launch_pair<decode_any_kernel>(kAnyWarps * 32,
                                       kAnyWarps * 2 * Part::floats(kAnyHeads, kMaxHeadDim) * 4, p, kAnyHeads, kAnyTile, 0.f, st);
    if (p.D <= 64) return launch_tc_heads<64>(p, st);
    if (p.D <= 128) return launch_tc_heads<128>(p, st);
    return launch_tc_heads<256>(p, st);
}

cudaError_t read_decode_error(int clear, int* code, cudaStream_t st) {
    return read_error(&g_error, clear, code, st);
}

}  // namespace ragged
}  // namespace rkv
