// r97b_internal.h -- declarations shared by the .cu files of libr97b200.so (not part of the ABI).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/r97b.h"

namespace r97b {

constexpr int kEpiStoreBf16 = R97B_EPI_STORE_BF16;
constexpr int kEpiStoreF32 = R97B_EPI_STORE_F32;
constexpr int kEpiAtomicF32 = R97B_EPI_ATOMIC_F32;
constexpr int kEpiAtomicF32T = R97B_EPI_ATOMIC_F32T;
constexpr int kEpiSplitBf16 = R97B_EPI_SPLIT_BF16;
constexpr int kEpiSwiglu = R97B_EPI_SWIGLU;
constexpr int kEpiSwigluBwd = R97B_EPI_SWIGLU_BWD;

int gemm_run(const R97bGemm& g, cudaStream_t stream);
// A row-major bf16 matrix [outer, inner] (row stride `ld` elements) as a 2D TMA tensor map with a
// (box_inner, box_outer) box and the 128-byte swizzle (gemm_tc.cu).
bool make_map(CUtensorMap* map, const void* ptr, int64_t inner, int64_t outer, int64_t ld, int box_inner,
              int box_outer);
// Token-major head rows as a 3D TMA map (column, row of a 128-token block, block's first token) with a
// (64, box_rows, 1) box: the block at token t is (x, r, t), r < 128, row r of it being token t + r. The rows and
// the tokens step by the same stride, so a box that starts at a negative r is zero there: a block of n < 128 tokens
// is loaded from r = n - 128 and lies at the end of its tile, with zero rows -- never a neighbour's -- before it.
// For the rows before r = 0 the copy engine reads, and discards, other rows that the map claims; so it claims rows of
// the T tokens alone: r < claim (128, or fewer for blocks of that many tokens) from the tokens t <= T - claim on.
struct RowsExtent {
    int64_t cols, rows, blocks;
};
inline RowsExtent rows_extent(int64_t heads, int64_t head, int32_t D, int64_t T, int claim) {
    const int64_t rows = T < claim ? T : claim;
    return RowsExtent{(heads - 1) * head + D, rows, T - rows + 1};
}
// Whether the map that claims 128 rows holds the block at `tok`.
__host__ __device__ inline bool rows_map_has(int64_t tok, int64_t T) { return tok + 128 <= T; }
bool make_rows_map(CUtensorMap* map, const R97bHeadRows& r, int64_t heads, int32_t D, int64_t T, int claim, int box_rows);
int num_sms();
// Opts kernel `fn` into at least `bytes` of dynamic shared memory on the device that is current. The
// runtime keeps this attribute per device; it is raised (never lowered) per (kernel, device), under a lock;
// returns false when the runtime refuses it (capi.cu).
bool smem_opt_in(const void* fn, int bytes);
template <typename F>
inline bool smem_opt_in(F* fn, int bytes) {
    return smem_opt_in(reinterpret_cast<const void*>(fn), bytes);
}
int64_t gemm_workspace_bytes(const R97bGemm& g);
// Each tcgen05 translation unit's error word (sm100.cuh), read and cleared.
unsigned gemm_error_word();
unsigned attn_error_word();
unsigned attn_fwd_error_word();
unsigned gdn_error_word();
unsigned loss_error_word();
unsigned gemm_i8_error_word();
unsigned rope_error_word();
unsigned attn_packed_error_word();

// Whether token-major head rows (R97bHeadRows) follow the ABI's rules for `heads` rows of D a token.
inline bool head_rows_ok(const R97bHeadRows& r, int64_t heads, int32_t D) {
    if (!r.ptr || (reinterpret_cast<uintptr_t>(r.ptr) & 15) || heads < 1 || heads > 65536) return false;
    if (r.head % 8 || r.tok % 8 || r.head < D || r.head > (1 << 24)) return false;
    return r.tok >= (heads - 1) * r.head + D && r.tok <= (1 << 30);
}

inline cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }

// Counts this library's kernel launches (r97b_launch_count); `n` = the launches the caller just queued.
void add_launches(int n);

// Records the CUDA error behind an R97B_ELAUNCH (r97b_last_launch_error reads it).
void note_launch_error(cudaError_t e);

inline int launch_status(int n = 1) {
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
        note_launch_error(e);
        return R97B_ELAUNCH;
    }
    add_launches(n);
    return R97B_OK;
}

}  // namespace r97b
