// Decode attention of requests with different lengths over one page pool.
//
//   o[b, h] = sum_t w_t v_t / sum_t w_t,  w_t = exp(scale q[b, h] . k_t),
//   t in [start_b, len_b), k_t and v_t rows of kv head h / (Hq / Hkv)
//
// in one pass over K and V with a running maximum (in the exponent of two) and sum.
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
#include <math.h>

#include "rkv_common.cuh"
#include "rkv_kernels.h"
#include "rkv_ragged.h"
#include "rkv_sm100.cuh"

namespace rkv {
namespace ragged {

static __device__ int g_error;

constexpr int kCtas = 148;      // one persistent CTA per SM
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

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

// n runs of as nearly equal length as may be, the longer ones first: with q = units / n and
// x = units % n, run i starts at i q + min(i, x).
struct Deal {
    int64_t q, x;
    __device__ __forceinline__ Deal(int64_t units, int64_t n) {
        q = units < (1ll << 32) ? (int64_t)((uint32_t)units / (uint32_t)n) : units / n;
        x = units - q * n;
    }
    __device__ __forceinline__ int64_t start(int64_t i) const { return i * q + min(i, x); }
    // the run that holds a unit
    __device__ __forceinline__ int64_t of(int64_t unit) const {
        const int64_t longer = x * (q + 1);
        return unit < longer ? unit / (q + 1) : x + (unit - longer) / q;
    }
};

// A part of a segment in memory: HG x {maximum, sum}, then HG x D accumulators.
struct Part {
    float* at; int HG, D;
    __device__ float& top(int row) const { return at[2 * row]; }
    __device__ float& sum(int row) const { return at[2 * row + 1]; }
    __device__ float* acc(int row) const { return at + 2 * HG + row * D; }
};

// Workspace: for each CTA what the part at the end of its run belongs to, then two parts per
// CTA (of a segment that began before its run; of one that began in it and goes on), then one
// per warp (of a segment that began before the warp's run and ended in it).
struct Workspace {
    int4* open; float* base; int64_t stride; int HG, D;
    __host__ __device__ static int64_t bytes(int64_t warps, int64_t HG, int64_t D) {
        return kCtas * 16 + (2 * kCtas + kCtas * warps) * HG * (D + 2) * 4;
    }
    __device__ Workspace(const DecodeParams& p, int hg)
        : open(static_cast<int4*>(p.ws)), base(reinterpret_cast<float*>(open + kCtas)),
          stride((int64_t)hg * (p.D + 2)), HG(hg), D(p.D) {}
    __device__ Part cta(int c, int which) const { return Part{base + (2 * c + which) * stride, HG, D}; }
    __device__ Part warp(int64_t worker) const { return Part{base + (2 * kCtas + worker) * stride, HG, D}; }
};

// The runs of a CTA and of its warps.
struct Runs {
    int64_t total;          // units of all requests
    int64_t ctas;           // CTAs that have a run (one unit per warp at least)
    int64_t cta0, cta1;     // the CTA's run
    int64_t unit;           // first unit of the warp's run
    int64_t count;          // and its length
    int b; int64_t u;       // request of that unit, and its place in it
};

template <int TT, int NW>
__device__ __forceinline__ Runs find_runs(const DecodeParams& p, int64_t per_tile) {
    __shared__ int64_t warp_sums[NW];
    __shared__ int s_b[NW];
    __shared__ int64_t s_u[NW];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (p.B + NW * 32 - 1) / (NW * 32);
    const int b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) {
        int64_t f, l;
        range_of(p, b, &f, &l);
        mine += tiles_of<TT>(f, l) * per_tile;
    }
    int64_t x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    Runs r{};
    int64_t before = x - mine;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        if (w < warp) before += warp_sums[w];
        r.total += warp_sums[w];
    }
    r.ctas = max((int64_t)1, min((int64_t)gridDim.x, r.total / NW));
    if (blockIdx.x >= r.ctas) return r;
    const Deal deal(r.total, r.ctas);
    r.cta0 = deal.start(blockIdx.x);
    r.cta1 = deal.start(blockIdx.x + 1);
    const Deal own(r.cta1 - r.cta0, NW);
    r.unit = r.cta0 + own.start(warp);
    r.count = r.cta0 + own.start(warp + 1) - r.unit;
    // the threads whose requests hold the start of a warp's run walk them
    if (mine > 0 && before < r.cta1 && before + mine > r.cta0) {
        for (int w = 0; w < NW; ++w) {
            const int64_t u = r.cta0 + own.start(w);
            if (u < before || u >= before + mine) continue;
            int64_t at = before;
            for (int b = b0; b < b1; ++b) {
                int64_t f, l;
                range_of(p, b, &f, &l);
                const int64_t k = tiles_of<TT>(f, l) * per_tile;
                if (u < at + k) { s_b[w] = b; s_u[w] = u - at; break; }
                at += k;
            }
        }
    }
    __syncthreads();
    r.b = s_b[warp];
    r.u = s_u[warp];
    return r;
}

// What a warp leaves for the join: the part of a segment that began before its run (`head`), and
// of one that began in its run and goes on behind it (`tail`).  A part that is there at the end
// of the run is in shared memory, a head that ended before is in the workspace.
struct Left {
    int head, ends, spilled, head_b, head_seg;
    int tail, tail_b, tail_seg;
    int64_t rest;           // units of the last segment behind the run
};

// Joins the parts of a CTA's warps.  In the order of the warps, a tail, or the first head, starts
// a chain, the heads behind it belong to the same segment, and one that ends closes it.  For each
// chain, a thread per row weighs the parts, then all threads add them up, VEC elements at a time.
template <int NW, int HG, int VEC>
__device__ __forceinline__ void join_parts(const DecodeParams& p, const Runs& r, const Workspace& ws,
                                           const Left* left, float* parts, int64_t stride, int groups) {
    __shared__ float s_weight[NW][HG], s_scale[HG];
    const int G = p.Hq / p.Hkv;
    const int c = blockIdx.x;
    if (threadIdx.x == 0) ws.open[c] = make_int4(-1, 0, 0, 0);
    for (int i = 0; i < NW + 1; ++i) {
        // chain 0: the first head; chain w + 1: the tail of warp w
        const int w = i == 0 ? 0 : i - 1;
        if (i == 0 ? !left[0].head : !left[w].tail) continue;
        int z = w;                      // last warp of the chain
        bool closed = i == 0 && left[0].ends;
        for (int v = w + 1; v < NW && !closed; ++v) {
            if (!left[v].head) continue;    // an empty run
            z = v;
            closed = left[v].ends;
        }
        auto part = [&](int v) {
            const bool spilled = left[v].spilled && !(i > 0 && v == w);
            return spilled ? ws.warp((int64_t)c * NW + v) : Part{parts + v * stride, HG, p.D};
        };
        const int b = i ? left[w].tail_b : left[w].head_b;
        const int seg = i ? left[w].tail_seg : left[w].head_seg;
        const int hq0 = seg / groups * G + seg % groups * HG;
        const int ng = min(HG, G - seg % groups * HG);
        const bool whole = i > 0 && closed;
        const Part to = ws.cta(c, i > 0);
        __syncthreads();    // the weights of the chain before
        if (threadIdx.x < ng) {
            const int row = threadIdx.x;
            float top = -INFINITY;
            for (int v = w; v <= z; ++v)
                if (v == w || left[v].head) top = fmaxf(top, part(v).top(row));
            const float base = top == -INFINITY ? 0.f : top;
            float sum = 0.f;
            for (int v = w; v <= z; ++v) {
                if (v != w && !left[v].head) continue;
                const Part from = part(v);
                const float a = sm100::ex2(from.top(row) - base);
                s_weight[v][row] = a;
                sum += from.sum(row) * a;
            }
            s_scale[row] = !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
            if (!whole) { to.top(row) = top; to.sum(row) = sum; }
            else if (p.lse) p.lse[(int64_t)b * p.Hq + hq0 + row] = top * kLn2 + logf(sum);
        }
        __syncthreads();
        const int per_row = p.D / VEC;
        for (int e = threadIdx.x; e < ng * per_row; e += NW * 32) {
            const int row = e / per_row, d = (e - row * per_row) * VEC;
            float o[VEC];
#pragma unroll
            for (int x = 0; x < VEC; ++x) o[x] = 0.f;
            for (int v = w; v <= z; ++v) {
                if (v != w && !left[v].head) continue;
                const float a = s_weight[v][row];
                const float* from = part(v).acc(row) + d;
                if constexpr (VEC == 4) {
                    const float4 f = *reinterpret_cast<const float4*>(from);
                    o[0] += f.x * a; o[1] += f.y * a; o[2] += f.z * a; o[3] += f.w * a;
                } else {
                    o[0] += from[0] * a;
                }
            }
            if (whole) {
                const int64_t at = (int64_t)b * p.o_stride_b + (int64_t)(hq0 + row) * p.o_stride_h + d;
#pragma unroll
                for (int x = 0; x < VEC; ++x) store_elt(p.out, at + x, p.dtype, o[x] * s_scale[row]);
            } else {
#pragma unroll
                for (int x = 0; x < VEC; ++x) to.acc(row)[d + x] = o[x];
            }
        }
        if (i > 0 && !closed && threadIdx.x == 0) {
            const int64_t last = r.cta1 + left[z].rest - 1;
            ws.open[c] = make_int4(b, seg, (int)(Deal(r.total, r.ctas).of(last) - c), 0);
        }
    }
}

// Position in the row of units: request, segment (kv head, group of query heads), tile.
template <int TT>
struct Walk {
    int b, seg, tile, tiles, first, last;
    __device__ __forceinline__ void enter(const DecodeParams& p, int request) {
        int64_t f, l;
        range_of(p, request, &f, &l);
        b = request;
        first = (int)f;
        last = (int)l;
        tiles = (int)tiles_of<TT>(f, l);
    }
    __device__ __forceinline__ void next(const DecodeParams& p, int per_tile) {
        if (++tile < tiles) return;
        tile = 0;
        if (++seg < per_tile) return;
        seg = 0;
        if (b + 1 < p.B) enter(p, b + 1);
    }
    __device__ __forceinline__ int token0() const { return (first / TT + tile) * TT; }
};

// ------------------------------------------------------------------------------------------
// 16-bit types, on tensor cores.  One warp works alone: it copies its tiles (TT tokens of K and
// V) into a ring of STAGES buffers of its own with 16-byte asynchronous copies, row by row
// through the page table, and multiplies with m16n8k16 from there.
//   S = Q K^T: the rows of A are query heads (MH of them), the columns of B are tokens;
//   O = P V:   P stays in registers, since the accumulators of S have the layout of A.
// Rounding P to 16 bits alone would add an error as large as the output's own rounding, so P
// goes in as hi + lo, both 16-bit.  With up to 8 heads, rows 8..15 of A are free and hold lo:
// the second half of the sum costs no instruction.  In fp16 the weights are scaled by 2^14
// (kBias), so that small ones do not fall below fp16's range; the scale is part of the maximum
// that is kept, and cancels.
// Rows outside the request's range are filled with zeros without being read: what the pool
// holds there (NaN included) never enters a product.
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool on) {
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

template <int DP, int TT, int NW, int STAGES>
struct TcShape {
    static constexpr int kPitch = DP * 2 + 16;          // odd in 16-byte units: no bank conflicts
    static constexpr int kPlane = TT * kPitch;          // K or V of a tile
    static constexpr int kStage = 2 * kPlane;
    static constexpr int kSmem = NW * STAGES * kStage;
};

template <bool kBf16, int DP, int MH, int TT, int NW, int STAGES>
__global__ void __launch_bounds__(NW * 32, 1)
decode_tc_kernel(DecodeParams p, int groups) {
    using Shape = TcShape<DP, TT, NW, STAGES>;
    static_assert(TT % 16 == 0 && TT <= 32 && DP % 16 == 0 && (MH == 8 || MH == 16), "shape");
    extern __shared__ __align__(128) char smem[];
    __shared__ Left left[NW];
    constexpr int kChunks = DP / 8;             // 16-byte chunks per row
    constexpr int kCopies = TT * kChunks / 32;  // copies per lane for K, and for V
    static_assert(TT * kChunks % 32 == 0, "a tile is a whole number of copies per lane");
    static_assert(STAGES * Shape::kStage >= MH * (DP + 2) * 4, "a part fits the warp's ring");
    constexpr float kBias = kBf16 ? 0.f : 14.f;
    constexpr int kRows = MH / 8;               // heads per lane: g, and g + 8
    constexpr int kQ = 2 * kRows;
    // the next segment's queries are fetched a tile ahead where registers allow
    constexpr bool kFetchQ = DP * MH <= 2048;
    sm100::grid_launch_dependents();
    sm100::grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per_tile = p.Hkv * groups;
    const int G = p.Hq / p.Hkv;
    const Workspace ws(p, MH);

    const Runs runs = find_runs<TT, NW>(p, per_tile);
    if (blockIdx.x >= runs.ctas) {
        if (threadIdx.x == 0) ws.open[blockIdx.x] = make_int4(-1, 0, 0, 0);
        return;
    }
    const uint32_t ring = sm100::smem_u32(smem) + warp * STAGES * Shape::kStage;
    const float scale2 = p.scale * kLog2e;
    Left mine{};
    if (runs.count > 0) {
        const int count = (int)runs.count;
        Walk<TT> put, get, nx;
        put.enter(p, runs.b);
        put.seg = (int)(runs.u / put.tiles);
        put.tile = (int)(runs.u % put.tiles);
        get = put;

        // ---- loads: lane r looks up row r of the tile; its page id is fetched a tile ahead
        int ahead = count;
        const int P = (int)p.P;
        auto fetch_page = [&]() -> int64_t {
            const int t = put.token0() + lane;
            return lane < TT && t >= put.first && t < put.last
                       ? p.table[(int64_t)put.b * p.table_stride + t / P] : -1;
        };
        int64_t page = fetch_page();
        const char* kbytes = static_cast<const char*>(p.k);
        const char* vbytes = static_cast<const char*>(p.v);
        auto issue = [&](int stage) {
            if (ahead > 0) {
                const int t = put.token0() + lane;
                int64_t row = -1;
                if (lane < TT && t >= put.first && t < put.last) {
                    if (page < 0 || page >= p.num_slots) { atomicMax(&g_error, kErrPage); page = 0; }
                    row = (page * p.stride_p + (int64_t)(t % P) * p.stride_t +
                           (int64_t)(put.seg / groups) * p.stride_h) * 2;
                }
                const uint32_t dst = ring + stage * Shape::kStage;
#pragma unroll
                for (int j = 0; j < kCopies; ++j) {
                    const int i = lane + 32 * j, r = i / kChunks, c = i % kChunks;
                    const int64_t off = __shfl_sync(0xffffffffu, row, r);
                    const bool on = off >= 0 && c * 8 < p.D;
                    const int64_t src = on ? off + c * 16 : 0;
                    copy16(dst + r * Shape::kPitch + c * 16, kbytes + src, on);
                    copy16(dst + Shape::kPlane + r * Shape::kPitch + c * 16, vbytes + src, on);
                }
                --ahead;
                put.next(p, per_tile);
                if (ahead > 0) page = fetch_page();
            }
            copies_commit();
        };

        // ---- products
        const int g = lane >> 2, c2 = (lane & 3) * 2;
        uint32_t q[DP / 16][kQ], qn[kFetchQ ? DP / 16 : 1][kQ];
        auto load_q = [&](const Walk<TT>& w, uint32_t (*to)[kQ]) {
            const int g0 = (w.seg % groups) * MH, ng = min(MH, G - g0);
            const char* qp = static_cast<const char*>(p.q) +
                             ((int64_t)w.b * p.q_stride_b +
                              (int64_t)(w.seg / groups * G + g0) * p.q_stride_h) * 2;
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
#pragma unroll
                for (int x = 0; x < kQ; ++x) {
                    const int r = g + (x % kRows) * 8, d = k * 16 + c2 + x / kRows * 8;
                    to[k][x] = r < ng && d < p.D
                                   ? *reinterpret_cast<const uint32_t*>(qp + (r * p.q_stride_h + d) * 2) : 0u;
                }
            }
        };
        load_q(get, q);
#pragma unroll
        for (int s = 0; s < STAGES; ++s) issue(s);

        float o[DP / 8][4], m[kRows], l[kRows];
        auto reset = [&]() {
#pragma unroll
            for (int n = 0; n < DP / 8; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x) o[n][x] = 0.f;
#pragma unroll
            for (int r = 0; r < kRows; ++r) { m[r] = -INFINITY; l[r] = 0.f; }
        };
        reset();
        // ldmatrix rows of this lane: K (token, dim) as B, V (token, dim) transposed as B
        const uint32_t k_lane = ((lane & 7) + (lane >> 4) * 8) * Shape::kPitch + ((lane >> 3) & 1) * 16;
        const uint32_t v_lane = ((lane & 7) + ((lane >> 3) & 1) * 8) * Shape::kPitch + (lane >> 4) * 16;
        int tile_in = get.tile;     // the segment's first tile in this run
        int stage = 0;
        for (int i = 0; i < count; ++i) {
            nx = get;
            nx.next(p, per_tile);
            if constexpr (kFetchQ)
                if (i + 1 < count && nx.tile == 0) load_q(nx, qn);
            copies_wait<STAGES - 1>();
            __syncwarp();
            const uint32_t kt = ring + stage * Shape::kStage, vt = kt + Shape::kPlane;
            float s[TT / 8][4];
#pragma unroll
            for (int n = 0; n < TT / 8; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x) s[n][x] = 0.f;
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
#pragma unroll
                for (int n = 0; n < TT / 16; ++n) {
                    uint32_t b0, b1, b2, b3;
                    sm100::ldsm_x4(kt + k_lane + n * 16 * Shape::kPitch + k * 32, b0, b1, b2, b3);
                    if constexpr (MH == 16) {
                        sm100::mma_16816<kBf16>(s[2 * n], q[k][0], q[k][1], q[k][2], q[k][3], b0, b1);
                        sm100::mma_16816<kBf16>(s[2 * n + 1], q[k][0], q[k][1], q[k][2], q[k][3], b2, b3);
                    } else {
                        sm100::mma_16816<kBf16>(s[2 * n], q[k][0], 0u, q[k][1], 0u, b0, b1);
                        sm100::mma_16816<kBf16>(s[2 * n + 1], q[k][0], 0u, q[k][1], 0u, b2, b3);
                    }
                }
            }
            const int t0 = get.token0();
            const bool edge = t0 < get.first || t0 + TT > get.last;
            bool grew = false;
            float alpha[kRows];
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                float top = -INFINITY;
#pragma unroll
                for (int n = 0; n < TT / 8; ++n) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float v = s[n][2 * r + x] * scale2;
                        if (edge) {
                            const int t = t0 + n * 8 + c2 + x;
                            if (t < get.first || t >= get.last) v = -INFINITY;
                        }
                        s[n][2 * r + x] = v;
                        top = fmaxf(top, v);
                    }
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // a head without a finite logit so far keeps 0 as its base: 2^(-inf) = 0, no NaN
                const float mn = fmaxf(m[r], top - kBias);
                const float base = mn == -INFINITY ? 0.f : mn;
                alpha[r] = sm100::ex2(m[r] - base);
                grew = grew || mn > m[r];
                m[r] = mn;
                float sum = 0.f;
#pragma unroll
                for (int n = 0; n < TT / 8; ++n) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float w = sm100::ex2(s[n][2 * r + x] - base);
                        s[n][2 * r + x] = w;
                        sum += w;
                    }
                }
                l[r] = l[r] * alpha[r] + sum;
            }
            if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                for (int n = 0; n < DP / 8; ++n) {
                    o[n][0] *= alpha[0];
                    o[n][1] *= alpha[0];
                    o[n][2] *= alpha[kRows - 1];
                    o[n][3] *= alpha[kRows - 1];
                }
            }
#pragma unroll
            for (int n = 0; n < TT / 16; ++n) {
                uint32_t hi[2][kRows], lo[2][kRows];
#pragma unroll
                for (int y = 0; y < 2; ++y) {
#pragma unroll
                    for (int r = 0; r < kRows; ++r) {
                        const float w0 = s[2 * n + y][2 * r], w1 = s[2 * n + y][2 * r + 1];
                        hi[y][r] = pack16<kBf16>(w0, w1);
                        const float2 back = unpack16<kBf16>(hi[y][r]);
                        lo[y][r] = pack16<kBf16>(w0 - back.x, w1 - back.y);
                    }
                }
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) {
                    uint32_t b0, b1, b2, b3;
                    sm100::ldsm_x4_trans(vt + v_lane + n * 16 * Shape::kPitch + d * 32, b0, b1, b2, b3);
                    if constexpr (MH == 16) {
                        sm100::mma_16816<kBf16>(o[2 * d], hi[0][0], hi[0][1], hi[1][0], hi[1][1], b0, b1);
                        sm100::mma_16816<kBf16>(o[2 * d + 1], hi[0][0], hi[0][1], hi[1][0], hi[1][1], b2, b3);
                        sm100::mma_16816<kBf16>(o[2 * d], lo[0][0], lo[0][1], lo[1][0], lo[1][1], b0, b1);
                        sm100::mma_16816<kBf16>(o[2 * d + 1], lo[0][0], lo[0][1], lo[1][0], lo[1][1], b2, b3);
                    } else {
                        sm100::mma_16816<kBf16>(o[2 * d], hi[0][0], lo[0][0], hi[1][0], lo[1][0], b0, b1);
                        sm100::mma_16816<kBf16>(o[2 * d + 1], hi[0][0], lo[0][0], hi[1][0], lo[1][0], b2, b3);
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
                const int h = get.seg / groups, g0 = (get.seg % groups) * MH;
                const int ng = min(MH, G - g0);
                if (!whole) {
                    if (tile_in > 0) {
                        mine.head = 1; mine.ends = ends; mine.spilled = !last;
                        mine.head_b = get.b; mine.head_seg = get.seg;
                    } else {
                        mine.tail = 1; mine.tail_b = get.b; mine.tail_seg = get.seg;
                    }
                    mine.rest = get.tiles - get.tile - 1;
                }
                const Part part = last ? Part{reinterpret_cast<float*>(smem + warp * STAGES * Shape::kStage), MH, p.D}
                                       : ws.warp((int64_t)blockIdx.x * NW + warp);
                if (last) __syncwarp();
#pragma unroll
                for (int r = 0; r < kRows; ++r) {
                    float sum = l[r];
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                    const int row = g + 8 * r;
                    if (row >= ng) continue;
                    const int hq = h * G + g0 + row;
                    const float inv = sum == 0.f ? 0.f : 1.f / sum;
                    char* out = static_cast<char*>(p.out) +
                                ((int64_t)get.b * p.o_stride_b + (int64_t)hq * p.o_stride_h) * 2;
#pragma unroll
                    for (int n = 0; n < DP / 8; ++n) {
                        const int d = n * 8 + c2;
                        if (d >= p.D) break;
                        const float x = MH == 16 ? o[n][2 * r] : o[n][0] + o[n][2];
                        const float y = MH == 16 ? o[n][2 * r + 1] : o[n][1] + o[n][3];
                        if (whole) *reinterpret_cast<uint32_t*>(out + d * 2) = pack16<kBf16>(x * inv, y * inv);
                        else *reinterpret_cast<float2*>(part.acc(row) + d) = make_float2(x, y);
                    }
                    if (c2 == 0) {
                        if (!whole) { part.top(row) = m[r]; part.sum(row) = sum; }
                        else if (p.lse) p.lse[(int64_t)get.b * p.Hq + hq] = m[r] * kLn2 + logf(sum);
                    }
                }
                reset();
                tile_in = 0;
                if (!last) {
                    if constexpr (kFetchQ) {
#pragma unroll
                        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
                            for (int x = 0; x < kQ; ++x) q[k][x] = qn[k][x];
                    } else {
                        load_q(nx, q);
                    }
                }
            }
            get = nx;
        }
    }
    if (lane == 0) left[warp] = mine;
    __syncthreads();
    join_parts<NW, MH, 4>(p, runs, ws, left, reinterpret_cast<float*>(smem), STAGES * Shape::kStage / 4, groups);
}

// ------------------------------------------------------------------------------------------
// Every other shape: any alignment, head_dim up to 256.  Lanes share the elements of a row; a
// token's logit is a sum over the warp.
// ------------------------------------------------------------------------------------------
constexpr int kAnyTile = 16, kAnyWarps = 8, kAnyHeads = 4;

__global__ void __launch_bounds__(kAnyWarps * 32)
decode_any_kernel(DecodeParams p, int groups) {
    constexpr int HG = kAnyHeads;
    __shared__ Left left[kAnyWarps];
    __shared__ float parts[kAnyWarps][HG * (kMaxHeadDim + 2)];
    sm100::grid_launch_dependents();
    sm100::grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t per_tile = (int64_t)p.Hkv * groups;
    const Workspace ws(p, HG);
    const Runs runs = find_runs<kAnyTile, kAnyWarps>(p, per_tile);
    if (blockIdx.x >= runs.ctas) {
        if (threadIdx.x == 0) ws.open[blockIdx.x] = make_int4(-1, 0, 0, 0);
        return;
    }
    const int G = p.Hq / p.Hkv;
    const int ne = (p.D + 31) / 32;
    const float scale2 = p.scale * kLog2e;
    Left mine{};
    int b = runs.b;
    int64_t u = runs.u, todo = runs.count;
    while (todo > 0) {
        int64_t first, last;
        range_of(p, b, &first, &last);
        const int64_t tiles = tiles_of<kAnyTile>(first, last);
        const int64_t* table = p.table + (int64_t)b * p.table_stride;
        while (todo > 0 && u < tiles * per_tile) {
            const int64_t seg = u / tiles, tile0 = u - seg * tiles;
            const int64_t tile1 = min(tiles, tile0 + todo);
            const int h = (int)(seg / groups), g0 = (int)(seg % groups) * HG;
            const int ng = min(HG, G - g0);
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
                    s *= scale2;
                    const float mn = fmaxf(m[g], s);
                    const float base = mn == -INFINITY ? 0.f : mn;
                    const float alpha = sm100::ex2(m[g] - base), w = sm100::ex2(s - base);
                    m[g] = mn;
                    l[g] = l[g] * alpha + w;
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[g][i] = acc[g][i] * alpha + w * vr[i];
                }
            }
            todo -= tile1 - tile0;
            u += tile1 - tile0;
            const bool ends = tile1 == tiles, whole = tile0 == 0 && ends;
            if (!whole) {
                if (tile0 > 0) {
                    mine.head = 1; mine.ends = ends; mine.spilled = todo > 0;
                    mine.head_b = b; mine.head_seg = (int)seg;
                } else {
                    mine.tail = 1; mine.tail_b = b; mine.tail_seg = (int)seg;
                }
                mine.rest = tiles - tile1;
            }
            const Part part = todo == 0 ? Part{parts[warp], HG, p.D}
                                        : ws.warp((int64_t)blockIdx.x * kAnyWarps + warp);
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
                    else if (p.lse) p.lse[(int64_t)b * p.Hq + hq] = m[g] * kLn2 + logf(l[g]);
                }
            }
        }
        ++b;
        u = 0;
    }
    if (lane == 0) left[warp] = mine;
    __syncthreads();
    join_parts<kAnyWarps, kAnyHeads, 1>(p, runs, ws, left, parts[0], HG * (kMaxHeadDim + 2), groups);
}

// ------------------------------------------------------------------------------------------
// CTA (c, row): row `row` of the segment that goes on behind the run of decode CTA c, if one
// does: its part there and one part of each CTA behind.  Each warp sums every kMergeWarps-th
// part, and the warps' sums are added in order.
// ------------------------------------------------------------------------------------------
constexpr int kMergeWarps = 4;

__global__ void __launch_bounds__(kMergeWarps * 32)
merge_kernel(DecodeParams p, int groups, int HG) {
    __shared__ float s_top[kMergeWarps], s_sum[kMergeWarps], s_acc[kMergeWarps][kMaxHeadDim];
    sm100::grid_launch_dependents();
    sm100::grid_dependency_wait();
    const Workspace ws(p, HG);
    const int c = blockIdx.x, row = blockIdx.y;
    const int4 open = ws.open[c];
    if (open.x < 0) return;
    const int G = p.Hq / p.Hkv;
    const int b = open.x, h = open.y / groups, g0 = (open.y % groups) * HG, n = open.z + 1;
    if (g0 + row >= G) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float top = -INFINITY;
    for (int i = threadIdx.x; i < n; i += kMergeWarps * 32) top = fmaxf(top, ws.cta(c + i, i == 0).top(row));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) s_top[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kMergeWarps; ++w) top = fmaxf(top, s_top[w]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, acc[kMaxHeadDim / 32];
#pragma unroll
    for (int x = 0; x < kMaxHeadDim / 32; ++x) acc[x] = 0.f;
#pragma unroll 4
    for (int i = warp; i < n; i += kMergeWarps) {
        const Part part = ws.cta(c + i, i == 0);
        const float a = sm100::ex2(part.top(row) - base);
        sum += part.sum(row) * a;
        const float* from = part.acc(row);
#pragma unroll
        for (int x = 0; x < kMaxHeadDim / 32; ++x)
            if (lane + 32 * x < p.D) acc[x] += from[lane + 32 * x] * a;
    }
    if (lane == 0) s_sum[warp] = sum;
#pragma unroll
    for (int x = 0; x < kMaxHeadDim / 32; ++x) s_acc[warp][lane + 32 * x] = acc[x];
    __syncthreads();
    float L = 0.f;
#pragma unroll
    for (int w = 0; w < kMergeWarps; ++w) L += s_sum[w];
    const int hq = h * G + g0 + row;
    for (int d = threadIdx.x; d < p.D; d += kMergeWarps * 32) {
        float o = 0.f;
#pragma unroll
        for (int w = 0; w < kMergeWarps; ++w) o += s_acc[w][d];
        store_elt(p.out, (int64_t)b * p.o_stride_b + (int64_t)hq * p.o_stride_h + d, p.dtype,
                  L == 0.f ? 0.f : o / L);
    }
    if (p.lse && threadIdx.x == 0) p.lse[(int64_t)b * p.Hq + hq] = top * kLn2 + logf(L);
}

namespace {

// 16-byte rows in the pool (its copies), 4-byte ones in q and out, token counts of 31 bits
bool tc_ok(const DecodeParams& p) {
    if (p.dtype == RKV_F32 || p.D % 8) return false;
    if (p.W * p.P > 0x7fffff00 || p.P > 0x7fffffff) return false;
    for (int64_t s : {p.stride_h, p.stride_p, p.stride_t})
        if (s % 8) return false;
    for (const void* ptr : {p.k, p.v})
        if (reinterpret_cast<uintptr_t>(ptr) & 15) return false;
    for (int64_t s : {p.q_stride_b, p.q_stride_h, p.o_stride_b, p.o_stride_h})
        if (s % 2) return false;
    return !((reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.out)) & 3);
}

// A decode kernel and its merge, each launched so that its start overlaps the end of the kernel
// before it (both wait for that kernel's results first).
template <typename Kernel>
cudaError_t launch_pair(Kernel kernel, int threads, int smem, const DecodeParams& p, int HG, cudaStream_t st) {
    const int groups = (p.Hq / p.Hkv + HG - 1) / HG;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
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
    cudaError_t e = counted(cudaLaunchKernelEx(&cfg, kernel, p, groups), 1);
    if (e != cudaSuccess) return e;
    cfg.gridDim = dim3(kCtas, HG);
    cfg.blockDim = dim3(kMergeWarps * 32);
    cfg.dynamicSmemBytes = 0;
    return counted(cudaLaunchKernelEx(&cfg, merge_kernel, p, groups, HG), 1);
}

template <bool kBf16, int DP, int MH>
cudaError_t launch_tc(const DecodeParams& p, cudaStream_t st) {
    constexpr int TT = DP <= 64 ? 32 : 16, NW = 8, STAGES = DP <= 128 ? 3 : 2 - (DP > 192);
    using Shape = TcShape<DP, TT, NW, STAGES>;
    static_assert(Shape::kSmem <= 232448 - 2048, "shared memory");
    return launch_pair(decode_tc_kernel<kBf16, DP, MH, TT, NW, STAGES>, NW * 32, Shape::kSmem, p, MH, st);
}

template <int DP>
cudaError_t launch_tc_dim(const DecodeParams& p, cudaStream_t st) {
    const bool wide = p.Hq / p.Hkv > 8;
    if (p.dtype == RKV_BF16) return wide ? launch_tc<true, DP, 16>(p, st) : launch_tc<true, DP, 8>(p, st);
    return wide ? launch_tc<false, DP, 16>(p, st) : launch_tc<false, DP, 8>(p, st);
}

}  // namespace

// Upper bound over the kernels that a call of these sizes may take.
size_t decode_workspace_bytes(int64_t Hq, int64_t Hkv, int64_t D) {
    return Workspace::bytes(8, Hq / Hkv > 8 ? 16 : 8, D);
}

cudaError_t launch_decode(const DecodeParams& p, cudaStream_t st) {
    if (!tc_ok(p)) return launch_pair(decode_any_kernel, kAnyWarps * 32, 0, p, kAnyHeads, st);
    if (p.D <= 64) return launch_tc_dim<64>(p, st);
    if (p.D <= 96) return launch_tc_dim<96>(p, st);
    if (p.D <= 128) return launch_tc_dim<128>(p, st);
    if (p.D <= 192) return launch_tc_dim<192>(p, st);
    return launch_tc_dim<256>(p, st);
}

cudaError_t read_decode_error(int clear, int* code) {
    cudaError_t e = cudaMemcpyFromSymbol(code, g_error, sizeof(int));
    if (e == cudaSuccess && clear && *code) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_error, &zero, sizeof(int));
    }
    return e;
}

}  // namespace ragged
}  // namespace rkv
