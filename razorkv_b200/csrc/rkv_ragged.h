// Parameter blocks and launchers of the ragged operators (requests of different lengths over
// one page pool).  Internal to the library.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace rkv {
namespace ragged {

// Codes of the ragged kernels' error word (the same numbers as the Python DEVICE_ERRORS).
constexpr int kErrPage = 2;      // a page or slot id outside the pool
constexpr int kErrLength = 3;    // a length outside [0, table capacity]
constexpr int kErrRefused = 4;   // a page-table step that could not be granted

// Division of 31-bit numbers by a divisor known at launch: the multiplicative inverse rounded up,
// 2^32 + mul = ceil(2^(32 + shift) / d) with 2^shift >= d, is exact below 2^31
// (Granlund and Montgomery, "Division by invariant integers using multiplication").
struct FastDiv {
    uint32_t mul = 0; int shift = 0;
    FastDiv() = default;
    explicit FastDiv(uint32_t d) {
        while ((1ull << shift) < d) ++shift;
        mul = (uint32_t)((((1ull << shift) - d) << 32) / d + 1);
    }
#ifdef __CUDACC__
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
        return (uint32_t)(((uint64_t)n * mul >> 32) + n >> shift);
    }
#endif
};

struct TableParams {
    const int64_t* lengths; const int64_t* new_lengths; int64_t R, P;
    int64_t* table; int64_t table_stride, W;
    int64_t* ring; int64_t C; int64_t* state;
    int64_t* out_lengths; int64_t* out_state;
    int64_t* slot_map; int64_t* positions; int64_t M; int64_t* starts;
    int in_place;               // an output is an input: written when every CTA has read it
    int narrow; FastDiv div_p;  // W * P below 2^31: division by P
};

struct AppendParams {
    void* k; void* v; int64_t stride_h, stride_p, stride_t, P, num_slots;
    const void* k_new; const void* v_new; int64_t new_stride_t, new_stride_h;
    int64_t T; const int64_t* slot_map; int Hkv, D, dtype;
    int narrow; FastDiv div_p;  // P below 2^31: division of such a slot by P
};

struct DecodeParams {
    const void* q; int64_t q_stride_b, q_stride_h;
    const void* k; const void* v; int64_t stride_h, stride_p, stride_t, P, num_slots;
    const int64_t* table; int64_t table_stride, W;
    const int64_t* lengths; const int64_t* starts;
    int B, Hq, Hkv, D, dtype;
    float scale;
    float bias;         // the kernel's weights are 2^bias times exp(scale * (q . k - base))
    void* out; int64_t o_stride_b, o_stride_h; float* lse;
    void* ws;
    FastDiv div_p;      // by P, where it is below 2^31
    int narrow;         // units of work are 31-bit numbers
};

cudaError_t launch_tables(const TableParams& p, cudaStream_t st);
cudaError_t launch_append(const AppendParams& p, cudaStream_t st);
size_t decode_workspace_bytes(int64_t Hq, int64_t Hkv, int64_t D);
cudaError_t launch_decode(const DecodeParams& p, cudaStream_t st);

// Reads (and with clear resets) the error word of one translation unit on the current device, in
// the stream's order, and waits for that.
cudaError_t read_table_error(int clear, int* code, cudaStream_t st);
cudaError_t read_decode_error(int clear, int* code, cudaStream_t st);

#ifdef __CUDACC__
// The above for one word.  It is reset only where it is still the code that was read: a larger one
// that another stream's kernel has set since is for the next caller.
static __global__ void clear_error_kernel(int* word, int code) { atomicCAS(word, code, 0); }

inline cudaError_t read_error(const void* symbol, int clear, int* code, cudaStream_t st) {
    void* word = nullptr;
    cudaError_t e = cudaGetSymbolAddress(&word, symbol);
    if (e == cudaSuccess) e = cudaMemcpyAsync(code, word, sizeof(int), cudaMemcpyDeviceToHost, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
    if (e != cudaSuccess || !clear || !*code) return e;
    clear_error_kernel<<<1, 1, 0, st>>>(static_cast<int*>(word), *code);
    e = cudaGetLastError();
    return e == cudaSuccess ? cudaStreamSynchronize(st) : e;
}
#endif

}  // namespace ragged
}  // namespace rkv
