// Page tables, slot map and append of requests that share one page pool.
//
// Both kernels move bytes and compute nothing: at decode steps (a token per request) they are
// bound by launch and memory latency, at prompts by writes.
#include "rkv_common.cuh"
#include "rkv_kernels.h"
#include "rkv_ragged.h"

namespace rkv {
namespace ragged {

static __device__ int g_error;

// ------------------------------------------------------------------------------------------
// Page tables.  Request r holds n_r tokens and is to hold m_r.  With pages(x) = ceil(x / P)
//   need_r = max(0, pages(m) - pages(n)),  give_r = max(0, pages(n) - pages(m)),
//   new_r  = max(0, m - n),
// and a, g, s their exclusive prefix sums over r, page j of request r comes from
// ring[(head + a_r + j - pages(n)) mod C] and page j given back goes to
// ring[(head + count + g_r + j - pages(m)) mod C].  Pages are taken from the ring's head and
// given back behind its tail, so what is read and what is written never overlap and no order
// between CTAs is needed; a stack would hand out the pages that the same call gives back.
//
// Every CTA sums need, give and new over all requests (16 bytes each, from L2) instead of
// waiting for another CTA's sums, then fills chunks of kChunk slot-map entries (one thread
// per entry) and of kChunk returned pages.  A chunk finds the request of each entry from
// marks: the thread that owns a request marks the entry where it starts, and a running
// maximum over the chunk carries the mark to the entries behind it.
// The state may be updated in place: it is written by the last CTA to finish, after every CTA
// has read it (a ticket in the state's third word, which returns to zero).
// ------------------------------------------------------------------------------------------
constexpr int kThreads = 1024;
constexpr int kChunk = kThreads;

struct Sums {
    int64_t need, give, fresh;
};

__device__ __forceinline__ int64_t shfl_up64(int64_t v, int o) {
    return __shfl_up_sync(0xffffffffu, v, o);
}

// Exclusive block-wide sums of three values and their totals.
__device__ Sums block_sums(Sums v, Sums* total, Sums* warp_sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Sums x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t a = shfl_up64(x.need, o), b = shfl_up64(x.give, o), c = shfl_up64(x.fresh, o);
        if (lane >= o) { x.need += a; x.give += b; x.fresh += c; }
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
        Sums w = warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t a = shfl_up64(w.need, o), b = shfl_up64(w.give, o), c = shfl_up64(w.fresh, o);
            if (lane >= o) { w.need += a; w.give += b; w.fresh += c; }
        }
        warp_sums[lane] = w;
    }
    __syncthreads();
    *total = warp_sums[31];
    if (warp > 0) {
        const Sums w = warp_sums[warp - 1];
        x.need += w.need; x.give += w.give; x.fresh += w.fresh;
    }
    return Sums{x.need - v.need, x.give - v.give, x.fresh - v.fresh};
}

// Running maximum over the block of one value per thread (values >= -1).
__device__ int block_running_max(int v, int* warp_max) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v = max(v, y);
    }
    if (lane == 31) warp_max[warp] = v;
    __syncthreads();
    int before = -1;
    for (int w = 0; w < warp; ++w) before = max(before, warp_max[w]);
    return max(v, before);
}

__global__ void __launch_bounds__(kThreads)
tables_kernel(TableParams p) {
    __shared__ Sums warp_sums[32];
    __shared__ int warp_max[32];
    __shared__ int mark[kChunk];           // entry at which a request starts, or -1
    __shared__ int64_t mark_req[kChunk], mark_at[kChunk], mark_pages[kChunk];
    __shared__ int s_last;
    const int tid = threadIdx.x;
    const int64_t head = p.state[0], count = p.state[1];
    const int64_t capacity = p.W * p.P;
    const int64_t per = (p.R + kThreads - 1) / kThreads;
    const int64_t r0 = min(p.R, tid * per), r1 = min(p.R, r0 + per);

    Sums mine{0, 0, 0};
    int bad = head < 0 || head >= p.C || count < 0 || count > p.C;
    for (int64_t r = r0; r < r1; ++r) {
        const int64_t n = p.lengths[r], m = p.new_lengths[r];
        if (n < 0 || n > capacity || m < 0 || m > capacity) { bad = 1; continue; }
        const int64_t have = (n + p.P - 1) / p.P, want = (m + p.P - 1) / p.P;
        mine.need += max((int64_t)0, want - have);
        mine.give += max((int64_t)0, have - want);
        mine.fresh += max((int64_t)0, m - n);
    }
    bad = __syncthreads_or(bad);
    Sums total;
    const Sums base = block_sums(mine, &total, warp_sums);
    // granted as a whole or not at all
    const bool ok = !bad && total.need <= count && total.fresh <= p.M &&
                    count - total.need + total.give <= p.C;

    // slot map, positions and new table entries
    for (int64_t c0 = (int64_t)blockIdx.x * kChunk; c0 < p.M; c0 += (int64_t)gridDim.x * kChunk) {
        const int64_t i = c0 + tid;
        if (!ok || c0 >= total.fresh) {
            if (i < p.M) { p.slot_map[i] = -1; p.positions[i] = 0; }
            continue;
        }
        __syncthreads();
        mark[tid] = -1;
        __syncthreads();
        if (base.fresh < c0 + kChunk && base.fresh + mine.fresh > c0) {
            int64_t s = base.fresh, a = base.need;
            for (int64_t r = r0; r < r1 && s < c0 + kChunk; ++r) {
                const int64_t n = p.lengths[r], m = p.new_lengths[r];
                if (m <= n) continue;
                if (s + (m - n) > c0) {
                    const int at = (int)max((int64_t)0, s - c0);
                    mark[at] = at;
                    mark_req[at] = r; mark_at[at] = s; mark_pages[at] = a;
                }
                s += m - n;
                a += max((int64_t)0, (m + p.P - 1) / p.P - (n + p.P - 1) / p.P);
            }
        }
        __syncthreads();
        const int at = block_running_max(mark[tid], warp_max);
        if (i >= p.M) continue;
        if (i >= total.fresh) { p.slot_map[i] = -1; p.positions[i] = 0; continue; }
        const int64_t r = mark_req[at];
        const int64_t n = p.lengths[r], t = n + (i - mark_at[at]);
        const int64_t j = t / p.P, off = t - j * p.P, have = (n + p.P - 1) / p.P;
        int64_t* entry = p.table + r * p.table_stride + j;
        const int64_t page = j < have ? *entry : p.ring[(head + mark_pages[at] + j - have) % p.C];
        const bool inside = page >= 0 && page < p.C;
        if (!inside) atomicMax(&g_error, kErrPage);
        if (j >= have && off == 0) *entry = page;
        p.slot_map[i] = inside ? page * p.P + off : -1;
        p.positions[i] = t;
    }

    // pages given back
    if (ok) {
        for (int64_t c0 = (int64_t)blockIdx.x * kChunk; c0 < total.give;
             c0 += (int64_t)gridDim.x * kChunk) {
            __syncthreads();
            mark[tid] = -1;
            __syncthreads();
            if (base.give < c0 + kChunk && base.give + mine.give > c0) {
                int64_t g = base.give;
                for (int64_t r = r0; r < r1 && g < c0 + kChunk; ++r) {
                    const int64_t have = (p.lengths[r] + p.P - 1) / p.P;
                    const int64_t want = (p.new_lengths[r] + p.P - 1) / p.P;
                    if (want >= have) continue;
                    if (g + (have - want) > c0) {
                        const int at = (int)max((int64_t)0, g - c0);
                        mark[at] = at;
                        mark_req[at] = r; mark_at[at] = g; mark_pages[at] = want;
                    }
                    g += have - want;
                }
            }
            __syncthreads();
            const int at = block_running_max(mark[tid], warp_max);
            const int64_t i = c0 + tid;
            if (i >= total.give) continue;
            p.ring[(head + count + i) % p.C] =
                p.table[mark_req[at] * p.table_stride + mark_pages[at] + (i - mark_at[at])];
        }
    }

    // token starts, lengths and state: the last CTA, so that they may replace the inputs
    if (gridDim.x > 1) {
        __syncthreads();
        if (tid == 0) {
            __threadfence();
            unsigned* ticket = reinterpret_cast<unsigned*>(p.state + 2);
            s_last = atomicInc(ticket, gridDim.x - 1) == gridDim.x - 1;
        }
        __syncthreads();
        if (!s_last) return;
    }
    __syncthreads();
    int64_t s = base.fresh;
    for (int64_t r = r0; r < r1; ++r) {
        const int64_t n = p.lengths[r], m = p.new_lengths[r];
        p.starts[r] = ok ? s : 0;
        p.out_lengths[r] = ok ? m : n;
        s += max((int64_t)0, m - n);
    }
    if (tid == 0) {
        p.starts[p.R] = ok ? total.fresh : 0;
        p.out_state[0] = ok ? (head + total.need) % p.C : head;
        p.out_state[1] = ok ? count - total.need + total.give : count;
        p.out_state[2] = 0;
        if (!ok) atomicMax(&g_error, kErrRefused);
    }
}

cudaError_t launch_tables(const TableParams& p, cudaStream_t st) {
    int64_t ctas = (p.M + kChunk - 1) / kChunk;
    if (ctas < 1) ctas = 1;
    if (ctas > 148) ctas = 148;
    tables_kernel<<<(unsigned)ctas, kThreads, 0, st>>>(p);
    return counted(cudaGetLastError(), 1);
}

// ------------------------------------------------------------------------------------------
// Append: row (t, h) of k_new / v_new to slot slot_map[t] of the pool.
// ------------------------------------------------------------------------------------------
template <typename Vec>
__global__ void __launch_bounds__(256)
append_kernel(AppendParams p, int chunks, int elts, int64_t tokens_per_cta) {
    const Vec* kn = static_cast<const Vec*>(p.k_new);
    const Vec* vn = static_cast<const Vec*>(p.v_new);
    Vec* k = static_cast<Vec*>(p.k);
    Vec* v = static_cast<Vec*>(p.v);
    const int64_t t0 = blockIdx.x * tokens_per_cta;
    const int per_token = p.Hkv * chunks;
    const int n = (int)min(tokens_per_cta, p.T - t0) * per_token;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int tl = i / per_token, rest = i - tl * per_token;
        const int h = rest / chunks, c = rest - h * chunks;
        const int64_t t = t0 + tl;
        const int64_t slot = p.slot_map[t];
        if (slot < 0) continue;
        const int64_t page = slot / p.P;
        if (page >= p.num_slots) { atomicMax(&g_error, kErrPage); continue; }
        const int64_t src = (t * p.new_stride_t + h * p.new_stride_h) / elts + c;
        const int64_t dst = (page * p.stride_p + (slot - page * p.P) * p.stride_t +
                             h * p.stride_h) / elts + c;
        k[dst] = kn[src];
        v[dst] = vn[src];
    }
}

cudaError_t launch_append(const AppendParams& p, cudaStream_t st) {
    if (p.T == 0) return cudaSuccess;
    const int eb = elt_bytes(p.dtype);
    bool vec = (p.D * eb) % 16 == 0;
    for (int64_t s : {p.stride_h, p.stride_p, p.stride_t, p.new_stride_t, p.new_stride_h})
        vec = vec && (s * eb) % 16 == 0;
    for (const void* ptr : {(const void*)p.k, (const void*)p.v, p.k_new, p.v_new})
        vec = vec && (reinterpret_cast<uintptr_t>(ptr) & 15) == 0;
    const int elts = vec ? 16 / eb : 1;
    const int chunks = p.D / elts;
    int64_t per = (1024 + p.Hkv * chunks - 1) / (p.Hkv * chunks);
    const int64_t ctas = (p.T + per - 1) / per;
    if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
    if (vec) append_kernel<uint4><<<(unsigned)ctas, 256, 0, st>>>(p, chunks, elts, per);
    else if (eb == 2) append_kernel<uint16_t><<<(unsigned)ctas, 256, 0, st>>>(p, chunks, elts, per);
    else append_kernel<uint32_t><<<(unsigned)ctas, 256, 0, st>>>(p, chunks, elts, per);
    return counted(cudaGetLastError(), 1);
}

cudaError_t read_table_error(int clear, int* code) {
    cudaError_t e = cudaMemcpyFromSymbol(code, g_error, sizeof(int));
    if (e == cudaSuccess && clear && *code) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_error, &zero, sizeof(int));
    }
    return e;
}

}  // namespace ragged
}  // namespace rkv
