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

constexpr int kTile = 16;       // tokens per unit
constexpr int kWarps = 8;       // warps per CTA
constexpr int kCtas = 148;
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
__device__ __forceinline__ int64_t tiles_of(int64_t first, int64_t last) {
    return last > first ? (last + kTile - 1) / kTile - first / kTile : 1;
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
    __device__ float* ml(int64_t worker, int which) const { return base + (worker * 2 + which) * stride; }
    __device__ float* acc(int64_t worker, int which) const { return ml(worker, which) + 2 * HG; }
};

template <int HG>
__global__ void __launch_bounds__(kWarps * 32)
decode_any_kernel(DecodeParams p, int groups) {
    __shared__ int64_t warp_sums[kWarps];
    __shared__ int64_t s_total;
    __shared__ int s_b[kWarps];
    __shared__ int64_t s_u[kWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t per_tile = (int64_t)p.Hkv * groups;
    int64_t* prefix = static_cast<int64_t*>(p.ws);

    // units before this thread's requests
    const int per = (p.B + blockDim.x - 1) / blockDim.x;
    const int b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) {
        int64_t f, l;
        range_of(p, b, &f, &l);
        mine += tiles_of(f, l) * per_tile;
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
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += warp_sums[w];
        total += warp_sums[w];
    }
    const int64_t workers = (int64_t)gridDim.x * kWarps;
    for (int w = 0; w < kWarps; ++w) {
        const int64_t u = run_start((int64_t)blockIdx.x * kWarps + w, workers, total);
        if (u >= before && u < before + mine) {
            int64_t at = before;
            for (int b = b0; b < b1; ++b) {
                int64_t f, l;
                range_of(p, b, &f, &l);
                const int64_t n = tiles_of(f, l) * per_tile;
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
            at += tiles_of(f, l) * per_tile;
        }
        if (tid == 0) prefix[p.B] = total;
    }
    __syncthreads();

    const int64_t worker = (int64_t)blockIdx.x * kWarps + warp;
    int64_t left = run_start(worker + 1, workers, total) - run_start(worker, workers, total);
    if (left == 0) return;
    const Fragments frag{reinterpret_cast<float*>(static_cast<char*>(p.ws) + prefix_bytes(p.B)),
                         (int64_t)HG * (p.D + 2), HG};
    const int G = p.Hq / p.Hkv;
    const int ne = (p.D + 31) / 32;
    const float scale2 = p.scale * kLog2e;
    int b = s_b[warp];
    int64_t u = s_u[warp];
    while (left > 0) {
        int64_t first, last;
        range_of(p, b, &first, &last);
        const int64_t tiles = tiles_of(first, last);
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

// One CTA per (request, query head): the fragments of its segment in the order of the tokens.
__global__ void __launch_bounds__(256)
merge_kernel(DecodeParams p, int groups, int HG, int64_t workers) {
    const int G = p.Hq / p.Hkv;
    const int b = blockIdx.x / p.Hq, hq = blockIdx.x % p.Hq;
    const int h = hq / G, gi = (hq % G) / HG, g = (hq % G) % HG;
    const int64_t* prefix = static_cast<const int64_t*>(p.ws);
    const int64_t total = prefix[p.B];
    const int64_t tiles = (prefix[b + 1] - prefix[b]) / ((int64_t)p.Hkv * groups);
    const int64_t u0 = prefix[b] + ((int64_t)h * groups + gi) * tiles, u1 = u0 + tiles;
    const int64_t w0 = run_of(u0, workers, total), w1 = run_of(u1 - 1, workers, total);
    if (w0 == w1) return;    // a warp had all of it
    const Fragments frag{reinterpret_cast<float*>(static_cast<char*>(p.ws) + prefix_bytes(p.B)),
                         (int64_t)HG * (p.D + 2), HG};
    float M = -INFINITY;
    for (int64_t w = w0; w <= w1; ++w) {
        const int64_t s = run_start(w, workers, total);
        if (s == run_start(w + 1, workers, total)) continue;
        M = fmaxf(M, frag.ml(w, w == w0 ? 1 : 0)[2 * g]);
    }
    const float base = M == -INFINITY ? 0.f : M;
    float L = 0.f, o = 0.f;
    for (int64_t w = w0; w <= w1; ++w) {
        const int64_t s = run_start(w, workers, total);
        if (s == run_start(w + 1, workers, total)) continue;
        const int which = w == w0 ? 1 : 0;
        const float a = sm100::ex2(frag.ml(w, which)[2 * g] - base);
        L += frag.ml(w, which)[2 * g + 1] * a;
        if (threadIdx.x < p.D) o += frag.acc(w, which)[g * p.D + threadIdx.x] * a;
    }
    if (threadIdx.x < p.D)
        store_elt(p.out, (int64_t)b * p.o_stride_b + (int64_t)hq * p.o_stride_h + threadIdx.x, p.dtype,
                  L == 0.f ? 0.f : o / L);
    if (p.lse && threadIdx.x == 0) p.lse[(int64_t)b * p.Hq + hq] = M * kLn2 + logf(L);
}

size_t decode_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D) {
    return prefix_bytes(B) + (size_t)kCtas * kWarps * 2 * 4 * (D + 2) * sizeof(float);
}

cudaError_t launch_decode(const DecodeParams& p, cudaStream_t st) {
    constexpr int HG = 4;
    const int groups = (p.Hq / p.Hkv + HG - 1) / HG;
    decode_any_kernel<HG><<<kCtas, kWarps * 32, 0, st>>>(p, groups);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    merge_kernel<<<(unsigned)((int64_t)p.B * p.Hq), 256, 0, st>>>(p, groups, HG, (int64_t)kCtas * kWarps);
    return counted(cudaGetLastError(), 2);
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
