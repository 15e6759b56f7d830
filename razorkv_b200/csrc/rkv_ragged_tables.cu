// Page tables, slot map and append of requests that share one page pool.
//
// Both kernels move bytes and compute nothing: at decode steps (a token per request) they are
// bound by launch and memory latency (tables of 64 requests 4.0 us, of 1024 with 25,000 new tokens
// 6.6, an append of 64 rows 1.8), long appends by memory.
#include "rkv_common.cuh"
#include "rkv_kernels.h"
#include "rkv_ragged.h"
#include "rkv_sm100.cuh"

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
// given back behind its tail, so with count + give <= C, which is checked, what is read and what is
// written never overlap and no order between CTAs is needed; a stack would hand out the pages that
// the same call gives back.
//
// Every CTA sums need, give and new over all requests (16 bytes each, from L2) instead of
// waiting for another CTA's sums, then fills chunks of kChunk slot-map entries (one thread
// per entry) and of kChunk returned pages.  A chunk finds the request of each entry from
// marks: the thread that owns a request marks the entry where it starts, and a running
// maximum over the chunk carries the mark to the entries behind it.
// The lengths and the state may be updated in place: then they are written by the last CTA to
// finish, after every CTA has read them (a ticket in the state's third word, which returns to
// zero); otherwise by the first CTA, without waiting.
// ------------------------------------------------------------------------------------------
constexpr int kThreads = 1024;
constexpr int kChunk = kThreads;

struct Sums {
    int64_t need, give, fresh;
};

// x / P for 0 <= x <= capacity, which is below 2^31 where the divisor is set
struct Pages {
    FastDiv div; int64_t P; bool narrow;
    __device__ __forceinline__ int64_t of(int64_t x) const { return narrow ? (int64_t)div((uint32_t)x) : x / P; }
    __device__ __forceinline__ int64_t up(int64_t x) const { return of(x) + (of(x) * P < x); }
};

// x mod C for 0 <= x < 3 C
__device__ __forceinline__ int64_t wrap(int64_t x, int64_t C) {
    x -= x >= C ? C : 0;
    return x - (x >= C ? C : 0);
}

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
    sm100::grid_launch_dependents();
    sm100::grid_dependency_wait();
    const int tid = threadIdx.x;
    const int64_t head = p.state[0], count = p.state[1];
    const int64_t capacity = p.W * p.P;
    const Pages pages{p.div_p, p.P, p.narrow != 0};
    const int64_t per = (p.R + kThreads - 1) / kThreads;
    const int64_t r0 = min(p.R, tid * per), r1 = min(p.R, r0 + per);

    Sums mine{0, 0, 0};
    int bad = head < 0 || head >= p.C || count < 0 || count > p.C;
    for (int64_t r = r0; r < r1; ++r) {
        const int64_t n = p.lengths[r], m = p.new_lengths[r];
        if (n < 0 || n > capacity || m < 0 || m > capacity) { bad = 1; continue; }
        const int64_t have = pages.up(n), want = pages.up(m);
        mine.need += max((int64_t)0, want - have);
        mine.give += max((int64_t)0, have - want);
        mine.fresh += max((int64_t)0, m - n);
    }
    bad = __syncthreads_or(bad);
    Sums total;
    const Sums base = block_sums(mine, &total, warp_sums);
    // granted as a whole or not at all
    const bool ok = !bad && total.need <= count && total.fresh <= p.M &&
                    count + total.give <= p.C;

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
                a += pages.up(m) - pages.up(n);
            }
        }
        __syncthreads();
        const int at = block_running_max(mark[tid], warp_max);
        if (i >= p.M) continue;
        if (i >= total.fresh) { p.slot_map[i] = -1; p.positions[i] = 0; continue; }
        const int64_t r = mark_req[at];
        const int64_t n = p.lengths[r], t = n + (i - mark_at[at]);
        const int64_t j = pages.of(t), off = t - j * p.P, have = pages.up(n);
        int64_t* entry = p.table + r * p.table_stride + j;
        const int64_t page = j < have ? *entry : p.ring[wrap(head + mark_pages[at] + j - have, p.C)];
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
                    const int64_t have = pages.up(p.lengths[r]), want = pages.up(p.new_lengths[r]);
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
            const int64_t page = p.table[mark_req[at] * p.table_stride + mark_pages[at] + (i - mark_at[at])];
            if (page < 0 || page >= p.C) atomicMax(&g_error, kErrPage);
            p.ring[wrap(head + count + i, p.C)] = page;
        }
    }

    // token starts, lengths and state
    if (!p.in_place) {
        if (blockIdx.x > 0) return;
    } else if (gridDim.x > 1) {
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
        p.out_state[0] = ok ? wrap(head + total.need, p.C) : head;
        p.out_state[1] = ok ? count - total.need + total.give : count;
        p.out_state[2] = 0;
        if (!ok) atomicMax(&g_error, kErrRefused);
    }
}

namespace {

// Launches so that the start overlaps the end of the kernel before, for whose results the kernel
// waits first.
template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), int64_t ctas, int threads, cudaStream_t st, const A&... args) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return counted(cudaLaunchKernelEx(&cfg, kernel, args...), 1);
}

}  // namespace

cudaError_t launch_tables(const TableParams& p, cudaStream_t st) {
    // a CTA per chunk of new tokens, or per 16 chunks of pages that may come back
    const double back = (double)p.R * (double)p.W / (16 * kChunk), fresh = ((double)p.M + kChunk - 1) / kChunk;
    const double ctas = back > fresh ? back : fresh;
    return launch(tables_kernel, ctas < 1 ? 1 : ctas > 148 ? 148 : (int64_t)ctas, kThreads, st, p);
}

// ------------------------------------------------------------------------------------------
// Append: row (t, h) of k_new / v_new to slot slot_map[t] of the pool, in pieces of a Vec.  A
// thread has kPieces pieces of K and of V on their way at a time.  A copy, bound by memory: for
// 32768 tokens of 8 heads x 128 fp16 (269 MB read and written), 128 threads of 2 pieces take
// 42.0 us (6.4 TB/s), 256 of 4 take 49.8, and with stores that stay in L2 44.3 and 51.7; 64
// tokens take 1.8 us and 2.8.
// ------------------------------------------------------------------------------------------
constexpr int kAppendThreads = 128, kPieces = 2;

template <typename Vec>
__global__ void __launch_bounds__(kAppendThreads)
append_kernel(AppendParams p, FastDiv div_token, FastDiv div_row, int per_token, int per_row, int elts,
              int tokens_per_cta) {
    sm100::grid_launch_dependents();
    sm100::grid_dependency_wait();
    const Vec* kn = static_cast<const Vec*>(p.k_new);
    const Vec* vn = static_cast<const Vec*>(p.v_new);
    Vec* k = static_cast<Vec*>(p.k);
    Vec* v = static_cast<Vec*>(p.v);
    const int64_t t0 = (int64_t)blockIdx.x * tokens_per_cta;
    const int n = (int)min((int64_t)tokens_per_cta, p.T - t0) * per_token;
    for (int i0 = threadIdx.x; i0 < n; i0 += kAppendThreads * kPieces) {
        int64_t slot[kPieces], src[kPieces];
        int in_row[kPieces], head[kPieces];
#pragma unroll
        for (int u = 0; u < kPieces; ++u) {
            const int i = i0 + u * kAppendThreads;
            const int tl = div_token(i), rest = i - tl * per_token;
            head[u] = div_row(rest);
            in_row[u] = rest - head[u] * per_row;
            const int64_t t = t0 + tl;
            slot[u] = i < n ? p.slot_map[t] : -1;
            src[u] = (t * p.new_stride_t + head[u] * p.new_stride_h) / elts + in_row[u];
        }
        Vec a[kPieces], b[kPieces];
#pragma unroll
        for (int u = 0; u < kPieces; ++u) {
            if (slot[u] < 0) continue;
            a[u] = __ldcs(kn + src[u]);
            b[u] = __ldcs(vn + src[u]);
        }
#pragma unroll
        for (int u = 0; u < kPieces; ++u) {
            if (slot[u] < 0) continue;
            const int64_t page = p.narrow && slot[u] < (1ll << 31) ? (int64_t)p.div_p((uint32_t)slot[u])
                                                                   : slot[u] / p.P;
            if (page >= p.num_slots) { atomicMax(&g_error, kErrPage); continue; }
            const int64_t dst = (page * p.stride_p + (slot[u] - page * p.P) * p.stride_t +
                                 head[u] * p.stride_h) / elts + in_row[u];
            __stcs(k + dst, a[u]);
            __stcs(v + dst, b[u]);
        }
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
    const int per_row = p.D / elts, per_token = p.Hkv * per_row;
    const int each = kAppendThreads * kPieces;
    const int tokens = per_token >= each ? 1 : each / per_token;
    const int64_t ctas = (p.T + tokens - 1) / tokens;
    if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
    const FastDiv dt((uint32_t)per_token), dr((uint32_t)per_row);
    if (vec) return launch(append_kernel<uint4>, ctas, kAppendThreads, st, p, dt, dr, per_token, per_row, elts, tokens);
    if (eb == 2) return launch(append_kernel<uint16_t>, ctas, kAppendThreads, st, p, dt, dr, per_token, per_row, elts, tokens);
    return launch(append_kernel<uint32_t>, ctas, kAppendThreads, st, p, dt, dr, per_token, per_row, elts, tokens);
}

cudaError_t read_table_error(int clear, int* code, cudaStream_t st) {
    return read_error(&g_error, clear, code, st);
}

}  // namespace ragged
}  // namespace rkv
