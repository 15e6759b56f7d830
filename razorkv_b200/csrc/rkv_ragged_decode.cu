// Decode attention of requests with different lengths over one page pool.
//
//   o[b, h] = sum_t w_t v_t / sum_t w_t,  w_t = exp(scale q[b, h] . k_t),
//   t in [start_b, len_b), k_t and v_t rows of kv head h / (Hq / Hkv)
//
// in one pass over K and V with a running maximum (in the exponent of two) and sum.
//
// Work is cut into units of kTile tokens of one (request, kv head, group of query heads); the
// units of all of them in a row are dealt out to the warps in equal contiguous runs, so a long
// request is split over many warps and short ones share one, whatever the lengths are.  They
// are only known on the device: every CTA sums the unit counts of all requests itself.  A run
// covers whole (request, kv head, group) segments, whose outputs the warp writes, and at most
// one unfinished segment at either end, whose (maximum, sum, accumulator) goes to the
// workspace; merge_kernel joins those in the order of the tokens, so results do not depend on
// timing.  The workspace needs no initial state.
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

// Start of worker w's run among `workers` equal runs of `units`, and the worker of a unit.
__device__ __forceinline__ int64_t run_start(int64_t w, int64_t workers, int64_t units) {
    return w * units / workers;
}
__device__ __forceinline__ int64_t run_of(int64_t unit, int64_t workers, int64_t units) {
    return ((unit + 1) * workers - 1) / units;
}

// Workspace: prefix[B + 1] of units (int64), then per worker two fragments (of a segment that
// began before the run, and of one that goes on behind it) of HG x {m, l} and HG x D floats.
__host__ __device__ inline int64_t prefix_bytes(int64_t B) { return ((B + 1) * 8 + 255) / 256 * 256; }

struct Fragments {
    float* base; int64_t stride; int HG;
    __device__ Fragments(const DecodeParams& p, int hg)
        : base(reinterpret_cast<float*>(static_cast<char*>(p.ws) + prefix_bytes(p.B))),
          stride((int64_t)hg * (p.D + 2)), HG(hg) {}
    __device__ float* ml(int64_t worker, int which) const { return base + (worker * 2 + which) * stride; }
    __device__ float* acc(int64_t worker, int which) const { return ml(worker, which) + 2 * HG; }
};

// The run of units of every warp of the CTA: request and unit within it, and the count.  Every
// CTA sums the unit counts of all requests; CTA 0 leaves their prefix sums to merge_kernel.
template <int TT, int NW>
__device__ __forceinline__ void find_runs(const DecodeParams& p, int64_t per_tile, int* b_out,
                                          int64_t* u_out, int64_t* left_out) {
    __shared__ int64_t warp_sums[NW];
    __shared__ int s_b[NW];
    __shared__ int64_t s_u[NW];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int64_t* prefix = static_cast<int64_t*>(p.ws);
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
    int64_t before = x - mine, total = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        if (w < warp) before += warp_sums[w];
        total += warp_sums[w];
    }
    const int64_t workers = (int64_t)gridDim.x * NW;
    // the threads whose requests hold a run's start walk them
    const int64_t lo = run_start((int64_t)blockIdx.x * NW, workers, total);
    const int64_t hi = run_start((int64_t)blockIdx.x * NW + NW - 1, workers, total);
    if (mine > 0 && before <= hi && before + mine > lo) {
        for (int w = 0; w < NW; ++w) {
            const int64_t u = run_start((int64_t)blockIdx.x * NW + w, workers, total);
            if (u < before || u >= before + mine) continue;
            int64_t at = before;
            for (int b = b0; b < b1; ++b) {
                int64_t f, l;
                range_of(p, b, &f, &l);
                const int64_t n = tiles_of<TT>(f, l) * per_tile;
                if (u < at + n) { s_b[w] = b; s_u[w] = u - at; break; }
                at += n;
            }
        }
    }
    if (blockIdx.x == 0) {
        int64_t at = before;
        for (int b = b0; b < b1; ++b) {
            int64_t f, l;
            range_of(p, b, &f, &l);
            prefix[b] = at;
            at += tiles_of<TT>(f, l) * per_tile;
        }
        if (tid == 0) prefix[p.B] = total;
    }
    __syncthreads();
    const int64_t worker = (int64_t)blockIdx.x * NW + warp;
    *left_out = run_start(worker + 1, workers, total) - run_start(worker, workers, total);
    *b_out = s_b[warp];
    *u_out = s_u[warp];
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
    constexpr int kChunks = DP / 8;             // 16-byte chunks per row
    constexpr int kCopies = TT * kChunks / 32;  // copies per lane for K, and for V
    static_assert(TT * kChunks % 32 == 0, "a tile is a whole number of copies per lane");
    constexpr float kBias = kBf16 ? 0.f : 14.f;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per_tile = p.Hkv * groups;
    const int G = p.Hq / p.Hkv;

    int b_start;
    int64_t u_start, count;
    find_runs<TT, NW>(p, per_tile, &b_start, &u_start, &count);
    if (count == 0) return;
    const int64_t worker = (int64_t)blockIdx.x * NW + warp;
    const uint32_t ring = sm100::smem_u32(smem) + warp * STAGES * Shape::kStage;
    const float scale2 = p.scale * kLog2e;

    Walk<TT> put, get;
    put.enter(p, b_start);
    put.seg = (int)(u_start / put.tiles);
    put.tile = (int)(u_start % put.tiles);
    get = put;

    // ---- loads: lane r looks up row r of the tile; its page id is fetched a tile ahead
    int64_t ahead = count;
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
#pragma unroll
    for (int s = 0; s < STAGES; ++s) issue(s);

    // ---- products
    const int g = lane >> 2, c2 = (lane & 3) * 2;
    uint32_t q[DP / 16][MH == 16 ? 4 : 2];
    float o[DP / 8][4];
    float m[2], l[2];
    constexpr int kRows = MH / 8;       // heads per lane: g, and g + 8
    const Fragments frag(p, MH);
    // ldmatrix rows of this lane: K (token, dim) as B, V (token, dim) transposed as B
    const uint32_t k_lane = ((lane & 7) + (lane >> 4) * 8) * Shape::kPitch + ((lane >> 3) & 1) * 16;
    const uint32_t v_lane = ((lane & 7) + ((lane >> 3) & 1) * 8) * Shape::kPitch + (lane >> 4) * 16;
    bool fresh = true;
    int tile_in = get.tile;     // first tile of the current segment that is this warp's
    int stage = 0;
    for (int64_t i = 0; i < count; ++i) {
        const int h = get.seg / groups, g0 = (get.seg % groups) * MH;
        const int ng = min(MH, G - g0);
        if (fresh) {
            fresh = false;
            tile_in = get.tile;
            const char* qp = static_cast<const char*>(p.q) +
                             ((int64_t)get.b * p.q_stride_b + (int64_t)(h * G + g0) * p.q_stride_h) * 2;
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
#pragma unroll
                for (int x = 0; x < (MH == 16 ? 4 : 2); ++x) {
                    const int r = MH == 16 ? g + (x & 1) * 8 : g;
                    const int d = k * 16 + c2 + (MH == 16 ? x >> 1 : x) * 8;
                    q[k][x] = r < ng && d < p.D
                                  ? *reinterpret_cast<const uint32_t*>(qp + (r * p.q_stride_h + d) * 2) : 0u;
                }
            }
#pragma unroll
            for (int n = 0; n < DP / 8; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x) o[n][x] = 0.f;
            m[0] = m[1] = -INFINITY;
            l[0] = l[1] = 0.f;
        }
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
        float alpha[2];
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
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
#pragma unroll
                for (int r = 0; r < kRows; ++r) {
                    const float w0 = s[2 * n + y][2 * r], w1 = s[2 * n + y][2 * r + 1];
                    hi[2 * y + r] = pack16<kBf16>(w0, w1);
                    const float2 back = unpack16<kBf16>(hi[2 * y + r]);
                    lo[2 * y + r] = pack16<kBf16>(w0 - back.x, w1 - back.y);
                }
            }
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                uint32_t b0, b1, b2, b3;
                sm100::ldsm_x4_trans(vt + v_lane + n * 16 * Shape::kPitch + d * 32, b0, b1, b2, b3);
                if constexpr (MH == 16) {
                    sm100::mma_16816<kBf16>(o[2 * d], hi[0], hi[1], hi[2], hi[3], b0, b1);
                    sm100::mma_16816<kBf16>(o[2 * d + 1], hi[0], hi[1], hi[2], hi[3], b2, b3);
                    sm100::mma_16816<kBf16>(o[2 * d], lo[0], lo[1], lo[2], lo[3], b0, b1);
                    sm100::mma_16816<kBf16>(o[2 * d + 1], lo[0], lo[1], lo[2], lo[3], b2, b3);
                } else {
                    sm100::mma_16816<kBf16>(o[2 * d], hi[0], lo[0], hi[2], lo[2], b0, b1);
                    sm100::mma_16816<kBf16>(o[2 * d + 1], hi[0], lo[0], hi[2], lo[2], b2, b3);
                }
            }
        }
        __syncwarp();
        issue(stage);
        stage = stage + 1 == STAGES ? 0 : stage + 1;

        // ---- the end of the segment, or of the run
        if (get.tile + 1 == get.tiles || i + 1 == count) {
            const bool whole = tile_in == 0 && get.tile + 1 == get.tiles;
            const int which = tile_in == 0 ? 1 : 0;
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                float sum = l[r];
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                const int row = g + 8 * r;
                if (row >= ng) continue;
                const int hq = h * G + g0 + row;
                float* part = frag.acc(worker, which) + row * p.D;
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
                    else *reinterpret_cast<float2*>(part + d) = make_float2(x, y);
                }
                if (c2 == 0) {
                    if (!whole) {
                        frag.ml(worker, which)[2 * row] = m[r];
                        frag.ml(worker, which)[2 * row + 1] = sum;
                    } else if (p.lse) {
                        p.lse[(int64_t)get.b * p.Hq + hq] = m[r] * kLn2 + logf(sum);
                    }
                }
            }
            fresh = true;
        }
        get.next(p, per_tile);
    }
}

// ------------------------------------------------------------------------------------------
// Every other shape: any alignment, head_dim up to 256, fp32 included.  Lanes share the
// elements of a row; a token's logit is a sum over the warp.
// ------------------------------------------------------------------------------------------
constexpr int kTile = 16;       // tokens per unit
constexpr int kWarps = 8;       // warps per CTA

template <int HG>
__global__ void __launch_bounds__(kWarps * 32)
decode_any_kernel(DecodeParams p, int groups) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t per_tile = (int64_t)p.Hkv * groups;
    int b;
    int64_t u, left;
    find_runs<kTile, kWarps>(p, per_tile, &b, &u, &left);
    if (left == 0) return;
    const int64_t worker = (int64_t)blockIdx.x * kWarps + warp;
    const Fragments frag(p, HG);
    const int G = p.Hq / p.Hkv;
    const int ne = (p.D + 31) / 32;
    const float scale2 = p.scale * kLog2e;
    while (left > 0) {
        int64_t first, last;
        range_of(p, b, &first, &last);
        const int64_t tiles = tiles_of<kTile>(first, last);
        const int64_t* table = p.table + (int64_t)b * p.table_stride;
        for (; left > 0 && u < tiles * per_tile;) {
            const int64_t seg = u / tiles, tile0 = u - seg * tiles;
            const int64_t tile1 = min(tiles, tile0 + left);
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
            const int64_t t1 = min(last, (first / kTile + tile1) * kTile);
            for (int64_t t = max(first, (first / kTile + tile0) * kTile); t < t1; ++t) {
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
            const bool whole = tile0 == 0 && tile1 == tiles;
            const int which = tile0 == 0 ? 1 : 0;
#pragma unroll
            for (int g = 0; g < HG; ++g) {
                if (g >= ng) break;
                const int hq = h * G + g0 + g;
                const float inv = l[g] == 0.f ? 0.f : 1.f / l[g];
                float* ml = frag.ml(worker, which) + 2 * g;
                float* part = frag.acc(worker, which) + g * p.D;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int e = lane + 32 * i;
                    if (e >= p.D) break;
                    if (whole)
                        store_elt(p.out, (int64_t)b * p.o_stride_b + (int64_t)hq * p.o_stride_h + e,
                                  p.dtype, acc[g][i] * inv);
                    else part[e] = acc[g][i];
                }
                if (lane == 0) {
                    if (!whole) { ml[0] = m[g]; ml[1] = l[g]; }
                    else if (p.lse) p.lse[(int64_t)b * p.Hq + hq] = m[g] * kLn2 + logf(l[g]);
                }
            }
            left -= tile1 - tile0;
            u += tile1 - tile0;
        }
        ++b;
        u = 0;
    }
}

// One CTA per (request, query head): the fragments of its segment.  Each warp sums every
// kMergeWarps-th fragment and the warps' sums are added in order.
constexpr int kMergeWarps = 8;

__global__ void __launch_bounds__(kMergeWarps * 32)
merge_kernel(DecodeParams p, int groups, int HG, int64_t workers) {
    __shared__ float s_top[kMergeWarps], s_sum[kMergeWarps], s_acc[kMergeWarps][kMaxHeadDim];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int G = p.Hq / p.Hkv;
    const int b = blockIdx.x / p.Hq, hq = blockIdx.x % p.Hq;
    const int h = hq / G, gi = (hq % G) / HG, g = (hq % G) % HG;
    const int64_t* prefix = static_cast<const int64_t*>(p.ws);
    const int64_t total = prefix[p.B];
    const int64_t tiles = (prefix[b + 1] - prefix[b]) / ((int64_t)p.Hkv * groups);
    const int64_t u0 = prefix[b] + ((int64_t)h * groups + gi) * tiles, u1 = u0 + tiles;
    const int64_t w0 = run_of(u0, workers, total), w1 = run_of(u1 - 1, workers, total);
    if (w0 == w1) return;    // a warp had all of it
    const Fragments frag(p, HG);
    // with fewer units than workers, some runs are empty and the others hold one unit
    const bool dense = total >= workers;
    const int n = (int)(dense ? w1 - w0 + 1 : tiles);
    auto fragment = [&](int i) {
        return frag.ml(dense ? w0 + i : run_of(u0 + i, workers, total), i == 0 ? 1 : 0);
    };
    float top = -INFINITY;
    for (int i = threadIdx.x; i < n; i += kMergeWarps * 32) top = fmaxf(top, fragment(i)[2 * g]);
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
    for (int i = warp; i < n; i += kMergeWarps) {
        const float* f = fragment(i);
        const float a = sm100::ex2(f[2 * g] - base);
        sum += f[2 * g + 1] * a;
#pragma unroll
        for (int x = 0; x < kMaxHeadDim / 32; ++x)
            if (lane + 32 * x < p.D) acc[x] += f[2 * HG + g * p.D + lane + 32 * x] * a;
    }
    if (lane == 0) s_sum[warp] = sum;
#pragma unroll
    for (int x = 0; x < kMaxHeadDim / 32; ++x) s_acc[warp][lane + 32 * x] = acc[x];
    __syncthreads();
    float L = 0.f;
#pragma unroll
    for (int w = 0; w < kMergeWarps; ++w) L += s_sum[w];
    for (int d = threadIdx.x; d < p.D; d += kMergeWarps * 32) {
        float o = 0.f;
#pragma unroll
        for (int w = 0; w < kMergeWarps; ++w) o += s_acc[w][d];
        store_elt(p.out, (int64_t)b * p.o_stride_b + (int64_t)hq * p.o_stride_h + d, p.dtype,
                  L == 0.f ? 0.f : o / L);
    }
    if (p.lse && threadIdx.x == 0) p.lse[(int64_t)b * p.Hq + hq] = top * kLn2 + logf(L);
}

size_t decode_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D) {
    return prefix_bytes(B) + (size_t)kCtas * kWarps * 2 * 16 * (D + 2) * sizeof(float);
}

namespace {

cudaError_t merge(const DecodeParams& p, int groups, int HG, int64_t workers, cudaStream_t st) {
    merge_kernel<<<(unsigned)((int64_t)p.B * p.Hq), kMergeWarps * 32, 0, st>>>(p, groups, HG, workers);
    return counted(cudaGetLastError(), 2);
}

template <bool kBf16, int DP, int MH>
cudaError_t launch_tc(const DecodeParams& p, cudaStream_t st) {
    constexpr int TT = DP <= 64 ? 32 : 16, NW = 8, STAGES = DP <= 128 ? 3 : 2 - (DP > 192);
    using Shape = TcShape<DP, TT, NW, STAGES>;
    static_assert(Shape::kSmem <= 232448, "shared memory");
    auto* kernel = decode_tc_kernel<kBf16, DP, MH, TT, NW, STAGES>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem);
    if (e != cudaSuccess) return e;
    const int groups = (p.Hq / p.Hkv + MH - 1) / MH;
    kernel<<<kCtas, NW * 32, Shape::kSmem, st>>>(p, groups);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    return merge(p, groups, MH, (int64_t)kCtas * NW, st);
}

template <int DP>
cudaError_t launch_tc_dim(const DecodeParams& p, cudaStream_t st) {
    const bool wide = p.Hq / p.Hkv > 8;
    if (p.dtype == RKV_BF16) return wide ? launch_tc<true, DP, 16>(p, st) : launch_tc<true, DP, 8>(p, st);
    return wide ? launch_tc<false, DP, 16>(p, st) : launch_tc<false, DP, 8>(p, st);
}

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

}  // namespace

cudaError_t launch_decode(const DecodeParams& p, cudaStream_t st) {
    if (tc_ok(p)) {
        if (p.D <= 64) return launch_tc_dim<64>(p, st);
        if (p.D <= 96) return launch_tc_dim<96>(p, st);
        if (p.D <= 128) return launch_tc_dim<128>(p, st);
        if (p.D <= 192) return launch_tc_dim<192>(p, st);
        return launch_tc_dim<256>(p, st);
    }
    constexpr int HG = 4;
    const int groups = (p.Hq / p.Hkv + HG - 1) / HG;
    decode_any_kernel<HG><<<kCtas, kWarps * 32, 0, st>>>(p, groups);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    return merge(p, groups, HG, (int64_t)kCtas * kWarps, st);
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
