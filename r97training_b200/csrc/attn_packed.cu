// attn_packed.cu -- causal grouped-query attention over packed (ragged) sequences, forward and the backward that
// recomputes the probabilities (reference: attention_twin and attention_host_adjoint,
// src/adjoint/host/attention.cpp:261-414).
//
//   o_t = sum_{j <= t} p_tj v_j,  p_tj = exp(scale q_t . k_j - lse_t)      over the tokens of t's own sequence
//   dv_j = sum_t p_tj do_t,  ds_tj = p_tj (do_t . v_j - do_t . o_t),  dq_t = scale sum_j ds_tj k_j,
//   dk_j = scale sum_t ds_tj q_t                                          (dk, dv summed over the group's heads)
//
// All products on tcgen05 with f32 accumulators in TMEM; P and dS are rounded to bf16 for the second products (half
// a bf16 step of each, what an output's own rounding costs), statistics and sums stay in f32.
//
// Blocks that end inside a tile sit at the tile's END, behind zero rows: the tensor maps address row r < 128 of the
// block that begins at token t as (column, r, t), token and row with one stride, and a box that starts at row n - 128
// has zeros before the block's first token. So no row of another sequence reaches a tile, nothing behind the last one
// is touched, and the same code serves every length. The maps claim the batch's own rows alone (the copy engine may
// read what they claim), which leaves out the blocks that begin in its last 127 tokens. A second map, which claims the
// last block's n tokens from each token on, holds that block and any other of n tokens at most; what is left (short
// sequences at the end, longer than the last one's last block) the producer warps copy themselves, 16 bytes a lane.
//
// What bounds it, measured a launch at a time at 2 x 4096 tokens of 16/4 heads of 256 (one sequence of 8192, 16/4 heads
// of 128): the forward 189-195 us (211-238) with the tensor pipe busy 80 % (64 %) of the cycles; the backward's passes
// 307 us dQ, 200 dV, 313 dK (276-297 dQ, 406-427 dK and dV) at 74, 84, 82 (76, 76) %. HBM takes 3-13 % of its rate
// throughout. A tile of dQ at D = 128, by the clock inside the kernel: 2040 cycles, of which the matrix unit works 1900
// on products that are 3 x 512 at its full rate (128-column products, both operands from shared memory at D = 128; with
// q and dO kept in tensor memory the tile took 1 % less, and units started later), and 130 pass between dS and the
// product that takes it. The exponentials take 980 of them beside the products; in the forward at D = 128 they take as
// long as its two products. A unit's start costs dQ two microseconds more: delta's loads and sums, before the first dS.
// In long runs the power limit sets the clock, and the time follows the products issued: 10 of 128 x 128 x D a tile at
// D = 256, forward and backward together (S formed four times), 9 at 128, where the mathematics needs 7.
#include "sm100.cuh"
#include "r97b_internal.h"
#include "fastmath.cuh"
#include "wmma16.cuh"

#include <algorithm>
#include <cuda_bf16.h>
#include <math.h>
#include <string.h>
#include <vector>

namespace r97b {

R97B_ERROR_READER(attn_packed_error_word)

namespace {

// ------------------------------------------------------------------------------------------ forward

constexpr int kBlk = 128;           // queries of a unit, keys of a tile
constexpr int kChunk = 16384;       // one ring stage
constexpr int kChunkLo = kChunk >> 4;               // and its step in a matrix descriptor
constexpr uint32_t kDescHi = sdesc_hi_sw128(1024);  // 8 rows of 128 bytes a swizzle atom
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr long long kWaitCycles = 4000000000ll;  // a wait's limit, about two seconds
constexpr float kLazy = 8.0f;       // log2 units a row's maximum may outgrow the reference before O is rescaled

// mbar_wait by every lane of a warp with one outcome for all: the warp stays converged, in the wait and when it gives up
// (a satisfied wait through divergent control flow costs 60 cycles more, a quarter of what a 16 KB chunk's products take).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
    uint32_t n = 0;
    long long t0 = 0;
    while (!__all_sync(0xFFFFFFFFu, mbar_try_wait(bar, parity))) {
        if ((++n & 255u) == 0) {
            const long long now = clock64();
            if (n == 256) t0 = now;
            const bool late = now - t0 > kWaitCycles;
            if (late) {
                atomicOr(&g_device_error, kErrTimeout);
                *abort = 1;
            }
            if (__any_sync(0xFFFFFFFFu, late || *abort != 0)) return false;
        }
    }
    return true;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&b);
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

template <int D>
struct FCfg {
    static constexpr int kBufs = D == 128 ? 3 : 2;       // S buffers, each with a softmax warpgroup of its own
    static constexpr int kThreads = 128 + 128 * kBufs;   // warps 0, 3: TMA, warp 1: MMA; the softmax warpgroups after
    static constexpr int kQBytes = kBlk * D * 2;
    static constexpr int kQStages = D == 128 ? 2 : 1;
    static constexpr int kStages = 9;
    static constexpr int kRingOff = kQStages * kQBytes;
    static constexpr int kBarOff = kRingOff + kStages * kChunk;
    static constexpr int kMaxOff = kBarOff + 768;        // float [kBufs][128]: the reference each buffer's tile used
    static constexpr int kFinOff = kMaxOff + kBufs * 512;  // float2 [2 (unit parity)][kBufs][128]: (reference, sum)
    static constexpr int kSmemBytes = kFinOff + 2 * kBufs * 1024 + 1024;
    static constexpr int kVRows = kChunk / (D * 2);      // keys of one V chunk
    static constexpr int kVLog2 = kVRows == 64 ? 6 : 5;
};

struct FwdArgs {
    const int4* blocks;
    __nv_bfloat16* o;
    float* lse;
    int64_t o_tok, o_head, ld_lse;
    int32_t Hq, grp, T;
    int32_t q_head, k_head, v_head;
    int32_t tail_n;                  // tokens of the batch's last block
    const __nv_bfloat16 *q, *k, *v;  // the operands again, for copy_chunk
    int64_t q_tok, k_tok, v_tok;
    float sl2;   // |scale| log2 e (1 for a scale of 0), so that the row maximum is the scores'
    float sign;  // of the scale: 1, -1 or 0
};

// Before the kernel ends on an abort: time for the copies and products still in flight, which nobody waits for any more,
// to land in this CTA's own memory (a bounded wait of about two milliseconds).
__device__ __forceinline__ void settle(const volatile int* abort) {
    if (!*abort) return;
    for (const long long t0 = clock64(); clock64() - t0 < 4000000;) __nanosleep(1000);
}

// By a whole warp: a chunk that TMA boxes of 2^log2_rows rows and 64 columns would fill (128-byte swizzle), the tile's rows
// from row0 on and, when those are not the whole tile, its further columns box by box. The block's tokens, the first at p with
// `tok` elements from one to the next, are the tile's rows from `shift` on; those before are zero.
__device__ __forceinline__ void copy_chunk(uint8_t* chunk, const __nv_bfloat16* p, int64_t tok, int log2_rows, int row0, int shift) {
#pragma unroll 2
    for (int k = threadIdx.x & 31; k < kChunk / 16; k += 32) {
        const int r = k >> 3, c = k & 7, t = row0 + (r & ((1 << log2_rows) - 1)) - shift;
        cp_async16(chunk + r * 128 + ((c ^ (r & 7)) << 4), p + (t >= 0 ? t : 0) * tok + (r >> log2_rows) * 64 + c * 8, t >= 0);
    }
}
// The warp's copies have landed and may be read by the tensor core: completes the barrier that a box's bytes would.
__device__ __forceinline__ void copies_done(uint64_t* bar, uint32_t lead) {
    cp_async_commit();
    cp_async_wait_all();
    fence_proxy_async_smem();
    __syncwarp();
    if (lead) mbar_arrive(bar);
}

// Which of an operand's two maps holds the block of n tokens at `tok`: 0, 1, or -1 for neither, which the warps copy. (Forward
// and backward of turns of 1, 9 and 130 tokens, 16/4 heads of 256, their last block copied: 67 us; by the second map: 49.)
__device__ __forceinline__ int map_of(int tok, int n, int T, int tail_n) {
    return rows_map_has(tok, T) ? 0 : (n <= tail_n ? 1 : -1);
}

struct Unit {
    int h, tok0, i, n;  // head, the block's first token, its index in the sequence, its tokens
};

// 32 accumulator values of each lane's row, times f, as 64 bytes of bf16 at p, for the rows from `shift` on. Four lanes trade
// 16-byte pieces first, so that they write a row's 64 bytes together: a store to 32 rows takes 32 cycles for its 32 lines. (2 x
// 4096 tokens, 16/4 heads of 256: forward 197 -> 189 us; a chat batch of 8192: forward 87 -> 80, dQ 133 -> 125.)
__device__ __forceinline__ void store_rows32(__nv_bfloat16* p, int64_t tok, int row, int shift, const uint32_t (&r)[32],
                                             float f) {
    uint32_t x[4][4];
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int k = 0; k < 4; ++k)
            x[v][k] = pack_bf16(__uint_as_float(r[v * 8 + k * 2]) * f, __uint_as_float(r[v * 8 + k * 2 + 1]) * f);
    const int a = threadIdx.x & 3;
#pragma unroll
    for (int bit = 1; bit <= 2; bit *= 2) {  // the 4 x 4 transpose, piece v of lane a for piece a of lane v
        const bool up = a & bit;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            if (v & bit) continue;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t got = __shfl_xor_sync(0xFFFFFFFFu, up ? x[v][k] : x[v + bit][k], bit);
                x[v][k] = up ? got : x[v][k];
                x[v + bit][k] = up ? x[v + bit][k] : got;
            }
        }
    }
    p += a * (8 - tok);
#pragma unroll
    for (int v = 0; v < 4; ++v)
        if (row - a + v >= shift)
            *reinterpret_cast<uint4*>(p + v * tok) = make_uint4(x[v][0], x[v][1], x[v][2], x[v][3]);
}

// The TMEM column of 16 consecutive k (k16-th) of a bf16 A operand whose writers own 32 f32 columns each and leave their
// values packed at the start of their own columns.
__device__ __forceinline__ constexpr int quarter_col(int k16) { return (k16 >> 1) * 32 + (k16 & 1) * 8; }

// The next unit of a CTA, for every role of it. The grid has one CTA a unit, longest units first; a CTA starts with its
// own and then takes over (cancels) the launch of the next one that has not started, so the units go to whichever SM is
// free. One role asks, as it loads the last tile of the unit before (asked a unit earlier, the key passes end with whole
// units waiting behind busy SMs); the answers pass through kSlots shared-memory slots, each read by every warp that walks
// the units (`readers` of them).
struct UnitQueue {
    static constexpr int kSlots = 4;
    uint4* slot;      // [kSlots]
    uint64_t* full;   // [kSlots]
    uint64_t* empty;  // [kSlots]
    volatile int* abort;

    __device__ void init(int readers) const {
        for (int i = 0; i < kSlots; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], readers);
        }
    }
    // Asks for the CTA's unit after its t-th (a whole warp, `lead` one lane of it); false when a wait gave up.
    __device__ bool ask(int t, uint32_t lead) const {
        const int i = t % kSlots;
        if (!warp_wait(&empty[i], (uint32_t)((t / kSlots) & 1) ^ 1u, abort)) return false;
        if (lead) {
            mbar_expect_tx(&full[i], 16);
            launch_cancel(&slot[i], &full[i]);
        }
        __syncwarp();
        return true;
    }
    // The unit after the t-th, or -1 when there is none (or a wait gave up): by a whole warp that counts as a reader.
    __device__ int next(int t) const {
        const int i = t % kSlots;
        if (!warp_wait(&full[i], (uint32_t)((t / kSlots) & 1), abort)) return -1;
        const int u = launch_cancelled(&slot[i]);
        fence_proxy_async_smem();  // the read, before the next answer's write
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(&empty[i]);
        return u;
    }
};

__device__ __forceinline__ Unit unit_geom(const int4* blocks, int heads, int u) {
    const int b = u / heads;
    const int4 e = blocks[b];
    return Unit{u - b * heads, e.x + e.z * kBlk, e.z, min(kBlk, e.y - e.z * kBlk)};
}

// One pass over the keys. A unit is one 128-query block of one head; key tile j of it: S_j = Q K_j^T into one of kBufs
// TMEM buffers, P_j = 2^(S_j c - m) as bf16 over the same buffer's columns, O += P_j V_j in TMEM. Each buffer has a
// softmax warpgroup, a thread a row, so the tiles' exponentials overlap one another and the products: S is issued kBufs - 1
// tiles ahead of P V, and P V starts on one half of the keys while the other's P is formed. The reference m a
// row's exponentials use is handed from tile to tile; it is moved (and O rescaled, by the threads that own the rows) only
// when the row's maximum has outgrown it by 2^8, which f32 sums and bf16 probabilities carry without loss. A unit's
// result is drained after the next unit's first P, which the tensor core has meanwhile been given the scores of.
// Three buffers at D = 128 (3 x 128 + 128 of the 512 TMEM columns), two at 256. Against two warpgroups in turn on two
// buffers with S a tile ahead inside a unit only: a chat batch of 16384 tokens, 8/2 heads of 128, 62 -> 49 us; 2 x 4096 tokens
// of 256, 213 -> 198. A softmax loop unrolled whole lost 100 us of the 540 at 12301 tokens to instruction fetches.
template <int D>
__global__ void __launch_bounds__(FCfg<D>::kThreads, 1)
    fwd_kernel(const __grid_constant__ CUtensorMap tQ, const __grid_constant__ CUtensorMap tK,
               const __grid_constant__ CUtensorMap tV, const __grid_constant__ CUtensorMap tQ1,
               const __grid_constant__ CUtensorMap tK1, const __grid_constant__ CUtensorMap tV1, const FwdArgs args) {
    using C = FCfg<D>;
    constexpr int ND = D / 64, NB = C::kBufs;
    constexpr int kVC = kBlk / C::kVRows;  // V chunks of a tile
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* ring = smem + C::kRingOff;
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
    const UnitQueue queue{reinterpret_cast<uint4*>(full_bar), full_bar + 8, full_bar + 12,
                          reinterpret_cast<volatile int*>(full_bar + 16)};
    volatile int* abort_flag = queue.abort;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(full_bar + 16) + 1;
    full_bar += 17;
    uint64_t* empty_bar = full_bar + C::kStages;
    uint64_t* q_full = empty_bar + C::kStages;  // [2]
    uint64_t* q_empty = q_full + 2;             // [2]
    uint64_t* s_full = q_empty + 2;             // [NB]
    uint64_t* p_full = s_full + NB;             // [NB][2]: P of keys 64 to 127, of 0 to 63 written
    uint64_t* pv_done = p_full + 2 * NB;        // [NB]
    uint64_t* o_full = pv_done + NB;
    uint64_t* o_empty = o_full + 1;
    uint64_t* max_bar = o_empty + 1;            // [NB][4]: a tile's reference written, by lane quarter
    uint64_t* fin_bar = max_bar + 4 * NB;       // [2][4]: the unit's sums written, by lane quarter
    float* ref_m = reinterpret_cast<float*>(smem + C::kMaxOff);
    float2* fin = reinterpret_cast<float2*>(smem + C::kFinOff);

    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0);
    const int lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        queue.init(3 + 4 * NB);
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&q_full[b], 2);
            mbar_init(&q_empty[b], 1);
        }
        for (int b = 0; b < NB; ++b) {
            mbar_init(&s_full[b], 1);
            mbar_init(&p_full[2 * b], 4);
            mbar_init(&p_full[2 * b + 1], 4);
            mbar_init(&pv_done[b], 1);
        }
        mbar_init(o_full, 1);
        mbar_init(o_empty, 4 * NB);
        for (int b = 0; b < 4 * NB; ++b) mbar_init(&max_bar[b], 1);
        for (int b = 0; b < 8; ++b) mbar_init(&fin_bar[b], NB);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch(&tQ);
        tma_prefetch(&tK);
        tma_prefetch(&tV);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_slot, 0);
    const uint32_t o_base = tmem + (uint32_t)(NB * kBlk);

    // Producers and MMA issuer walk the CTA's tiles with two cursors: S of a tile (and its K) NB - 1 tiles ahead of P V
    // (and its V), across the units' borders too, so that a unit's first softmax runs beside the last one's.
    if (warp == 0 || warp == 3) {
        // ------------------------------------------------------------- TMA producers: every other chunk each
        const uint32_t lead = elect_one();
        const int p = warp == 3;
        int stage = p;
        uint32_t phase = 0;
        bool ok = true;
        struct Cursor {
            int x, seq0, i, shift, j;
        };
        Cursor ahead{}, behind{}, w0{}, w1{};  // w0, w1: the units between, oldest first
        int waiting = 0, led = 0, lt = 0;
        bool more = true, fresh = true;  // a unit for `ahead`; its Q not loaded yet
        int u = blockIdx.x;
        // Rolled, and with one call for keys and values: the warps share an instruction cache, which a second copy of this (the
        // code for the batch's last blocks) overfilled (2 x 4096 tokens of 16/4 heads of 256: 229 -> 239 us back to back).
        auto load = [&](bool v, const Cursor& c) {
            const int tok = c.seq0 + c.j * kBlk, r0 = c.j == c.i ? -c.shift : 0;
            const int at = map_of(tok, kBlk + r0, args.T, args.tail_n);
            const CUtensorMap* map = v ? (at == 1 ? &tV1 : &tV) : (at == 1 ? &tK1 : &tK);
#pragma unroll 1
            for (int ch = p; ch < (v ? kVC : ND); ch += 2) {
                if (!(ok = warp_wait(&empty_bar[stage], phase ^ 1u, abort_flag))) return;
                uint8_t* st = ring + stage * kChunk;
                const int row0 = v ? (ch + kVC / 2) % kVC * C::kVRows : 0;  // keys 64 on first
                const int col = c.x * (v ? args.v_head : args.k_head) + (v ? 0 : 64 * ch);
                if (at < 0) {
                    const int64_t step = v ? args.v_tok : args.k_tok;
                    copy_chunk(st, (v ? args.v : args.k) + tok * step + col, step, v ? C::kVLog2 : 7, row0, -r0);
                    copies_done(&full_bar[stage], lead);
                } else if (lead) {
                    mbar_expect_tx(&full_bar[stage], kChunk);
                    tma_load_3d(st, map, &full_bar[stage], col, r0 + row0, tok);
                    if (v) {
#pragma unroll
                        for (int n = 1; n < ND; ++n)
                            tma_load_3d(st + n * (C::kVRows * 128), map, &full_bar[stage], col + 64 * n, r0 + row0, tok);
                    }
                }
                if ((stage += 2) >= C::kStages) {
                    stage -= C::kStages;
                    phase ^= 1u;
                }
            }
        };
        while (ok) {
            if (fresh) {  // the next unit, or none
                if (lt > 0) u = queue.next(lt - 1);
                fresh = false;
                more = u >= 0;
                if (more) {
                    const Unit un = unit_geom(args.blocks, args.Hq, u);
                    ahead = Cursor{un.h / args.grp, un.tok0 - un.i * kBlk, un.i, kBlk - un.n, 0};
                    const int qs = lt % C::kQStages;
                    if (!(ok = warp_wait(&q_empty[qs], (uint32_t)((lt / C::kQStages) & 1) ^ 1u, abort_flag))) break;
                    const int at = map_of(un.tok0, un.n, args.T, args.tail_n);
                    if (at < 0) {
#pragma unroll 1
                        for (int s = p; s < ND; s += 2)
                            copy_chunk(smem + qs * C::kQBytes + s * kChunk,
                                       args.q + un.tok0 * args.q_tok + un.h * args.q_head + 64 * s, args.q_tok, 7, 0, ahead.shift);
                        copies_done(&q_full[qs], lead);
                    } else if (lead) {
                        mbar_expect_tx(&q_full[qs], C::kQBytes / 2);
                        for (int s = p; s < ND; s += 2)
                            tma_load_3d(smem + qs * C::kQBytes + s * kChunk, at ? &tQ1 : &tQ, &q_full[qs], un.h * args.q_head + 64 * s,
                                        -ahead.shift, un.tok0);
                    }
                    if (waiting == 0) {
                        behind = ahead;
                    } else if (waiting == 1) {
                        w0 = ahead;
                    } else {
                        w1 = ahead;
                    }
                    ++waiting;
                    ++lt;
                }
            }
            if (!more && led == 0) break;
#pragma unroll 1
            for (int v = more ? 0 : 1; v < 2; ++v) {  // K of the tile ahead, V of the one behind
                if (!v && p && ahead.j == ahead.i && !(ok = queue.ask(lt - 1, lead))) break;
                load(v, v ? behind : ahead);
                if (!ok) break;
                if (!v) {
                    fresh = ++ahead.j > ahead.i;
                    if (++led < NB) break;
                } else {
                    --led;
                    if (++behind.j > behind.i) {
                        behind = w0, w0 = w1;
                        --waiting;
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------- MMA issuer
        const uint32_t lead = elect_one();
        constexpr uint32_t idesc_s = make_idesc_bf16(kBlk, kBlk, 0, 0);
        constexpr uint32_t idesc_o = make_idesc_bf16(kBlk, D, 0, 1);
        const uint32_t k_lo = sdesc_lo(smem_u32(ring), 16), v_lo = sdesc_lo(smem_u32(ring), C::kVRows * 128);
        int stage = 0, sb = 0, pb = 0;  // sb, pb: the next S's and the next P's buffer
        uint32_t phase = 0, p_phase = 0;
        bool ok = true;
        auto next = [&]() {
            umma_commit_by(lead, &empty_bar[stage]);
            if (++stage == C::kStages) {
                stage = 0;
                phase ^= 1u;
            }
        };
        int js = 0, ns = 0, jp = 0, np = 0, w0 = 0, w1 = 0;  // tile and tiles of the units at S and at P V; those between
        int waiting = 0, led = 0, lt = 0, lt_p = 0;
        uint32_t q_lo = 0;
        bool more = true, fresh = true;
        int u = blockIdx.x;
        while (ok) {
            if (fresh) {
                if (lt > 0) u = queue.next(lt - 1);
                fresh = false;
                more = u >= 0;
                if (more) {
                    ns = unit_geom(args.blocks, args.Hq, u).i + 1;
                    js = 0;
                    const int qs = lt % C::kQStages;
                    if (!(ok = warp_wait(&q_full[qs], (uint32_t)((lt / C::kQStages) & 1), abort_flag))) break;
                    q_lo = sdesc_lo(smem_u32(smem), 16) + (uint32_t)(qs * (C::kQBytes >> 4));
                    if (waiting == 0) {
                        np = ns;
                    } else if (waiting == 1) {
                        w0 = ns;
                    } else {
                        w1 = ns;
                    }
                    ++waiting;
                    ++lt;
                }
            }
            if (more) {
                // S into the buffer whose last P V is already before it in the issue order
#pragma unroll
                for (int kb = 0; kb < ND; ++kb) {
                    if (!(ok = ok && warp_wait(&full_bar[stage], phase, abort_flag))) break;
                    tc_fence_after();
                    const uint32_t a = q_lo + (uint32_t)(kb * kChunkLo), b = k_lo + (uint32_t)(stage * kChunkLo);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        umma_f16_by(lead, tmem + (uint32_t)(sb * kBlk), sdesc(a + kk * 2, kDescHi),
                                    sdesc(b + kk * 2, kDescHi), idesc_s, (kb > 0 || kk > 0) ? 1u : 0u);
                    next();
                }
                if (!ok) break;
                umma_commit_by(lead, &s_full[sb]);
                if (++sb == NB) sb = 0;
                if (++js == ns) {
                    umma_commit_by(lead, &q_empty[(lt - 1) % C::kQStages]);
                    fresh = true;
                }
                if (++led < NB) continue;
            }
            if (led == 0) break;
            if (jp == 0 && !(ok = warp_wait(o_empty, (uint32_t)(lt_p & 1) ^ 1u, abort_flag))) break;
#pragma unroll
            for (int ch = 0; ch < kVC; ++ch) {
                if (ch % (kVC / 2) == 0) ok = ok && warp_wait(&p_full[2 * pb + ch / (kVC / 2)], p_phase, abort_flag);
                if (!(ok = ok && warp_wait(&full_bar[stage], phase, abort_flag))) break;
                tc_fence_after();
                const uint32_t v = v_lo + (uint32_t)(stage * kChunkLo);
#pragma unroll
                for (int kk = 0; kk < C::kVRows / 16; ++kk)
                    umma_f16_ts_by(lead, o_base, tmem + (uint32_t)(pb * kBlk + 64 + (ch * C::kVRows + kk * 16) / 2),
                                   sdesc(v + kk * 128, kDescHi), idesc_o, (jp > 0 || ch > 0 || kk > 0) ? 1u : 0u);
                next();
            }
            if (!ok) break;
            umma_commit_by(lead, &pv_done[pb]);
            if (++pb == NB) {
                pb = 0;
                p_phase ^= 1u;
            }
            --led;
            if (++jp == np) {
                umma_commit_by(lead, o_full);
                ++lt_p;
                jp = 0;
                np = w0, w0 = w1;
                --waiting;
            }
        }
    } else if (warp >= 4) {
        // ------------------------------------------------------------- softmax
        const int q = warp & 3, w = (warp - 4) >> 2;
        const int row = q * 32 + lane;
        const uint32_t lane_off = (uint32_t)(q * 32) << 16;
        const uint32_t s_tmem = tmem + lane_off + (uint32_t)(w * kBlk), o_tmem = o_base + lane_off;
        const int prev = w == 0 ? NB - 1 : w - 1;  // the buffer of the tile before
        int turn = w;                              // tiles until this warpgroup's next
        uint32_t phase = 0;                        // of this buffer's barriers
        bool ok = true;
        // the unit whose result is still in TMEM: its number and geometry, the buffer of its last tile
        int d_lt = -1, d_last = 0, d_nt = 0, d_h = 0, d_shift = 0;
        int64_t d_tok = 0;
        auto drain = [&]() -> bool {
            const float2* sums = fin + (d_lt & 1) * (NB * 128);
            if (!warp_wait(&fin_bar[(d_lt & 1) * 4 + q], (uint32_t)((d_lt >> 1) & 1), abort_flag)) return false;
            // the row's sums, moved to the last tile's reference, the last tile's buffer first (which buffer that is
            // differs with the units a CTA has had before, the order of the sum does not)
            float m = sums[d_last * 128 + row].x;
            m = m == -INFINITY ? 0.0f : m;
            float sum = 0.0f;
#pragma unroll
            for (int back = 0, b = d_last; back < NB; ++back) {
                // a buffer that had no tile of the unit holds nothing of it
                const float2 s = sums[b * 128 + row];
                if (back < d_nt) sum = back == 0 ? s.y : fmaf(s.y, ex2_ftz(s.x - m), sum);
                b = b == 0 ? NB - 1 : b - 1;
            }
            if (!warp_wait(o_full, (uint32_t)(d_lt & 1), abort_flag)) return false;
            tc_fence_after();
            if (w == 0 && row >= d_shift) args.lse[d_h * args.ld_lse + d_tok] = fmaf(m, kLn2, logf(sum));
            const float inv = 1.0f / sum;
            __nv_bfloat16* op = args.o + d_tok * args.o_tok + d_h * args.o_head;
#pragma unroll 1
            for (int cc = w; cc < D / 32; cc += NB) {
                uint32_t r[32];
                __syncwarp();
                tmem_ld32(o_tmem + (uint32_t)(cc * 32), r);
                tmem_ld_wait();
                store_rows32(op + cc * 32, args.o_tok, row, d_shift, r, inv);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(o_empty);
            d_lt = -1;
            return true;
        };
        for (int u = blockIdx.x, lt = 0; ok && u >= 0; u = ok ? queue.next(lt) : -1, ++lt) {
            const Unit un = unit_geom(args.blocks, args.Hq, u);
            const int shift = kBlk - un.n, nt = un.i + 1;
            float m = 0.0f, l = 0.0f;  // the reference of this warpgroup's last tile, its tiles' sum relative to it
            int j = turn;
            for (; j < nt; j += NB) {
                if (!(ok = warp_wait(&s_full[w], phase, abort_flag))) break;
                tc_fence_after();
                const bool diag = j == un.i;
                float mx[2] = {-INFINITY, -INFINITY};
                float xa[32], xb[32];
                auto load = [&](float(&x)[32], int cc) {
                    tmem_ld32(s_tmem + (uint32_t)(cc * 32), *reinterpret_cast<uint32_t(*)[32]>(&x[0]));
                };
                // a chunk's part of the row maximum; a NaN score makes it NaN, and with it the row
                auto maximum = [&](const float(&x)[32]) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        mx[0] = max3_nan(mx[0], x[e], x[e + 1]);
                        mx[1] = max3_nan(mx[1], x[e + 2], x[e + 3]);
                    }
                };
                // Signs and masks are put into the buffer beforehand, a chunk at a time in one small loop: code for them
                // where the scores are used is fetched cold on every diagonal tile and cost more than this pass. On the
                // diagonal a warp's rows see the chunks before theirs whole.
                if (args.sign != 1.0f || diag) {
#pragma unroll 1
                    for (int cc = 0; cc < 4; ++cc) {
                        if (args.sign == 1.0f && cc < q && cc * 32 >= shift) continue;
                        load(xa, cc);
                        tmem_ld_wait();
                        const int hi = diag ? row - cc * 32 : 32, lo = diag ? shift - cc * 32 : 0;
                        const uint32_t upto = hi < 0 ? 0u : (hi >= 31 ? ~0u : (2u << hi) - 1u);
                        const uint32_t seen = upto & (lo <= 0 ? ~0u : (lo >= 32 ? 0u : ~0u << lo));
#pragma unroll
                        for (int e = 0; e < 32; ++e) xa[e] = seen & (1u << e) ? xa[e] * args.sign : -INFINITY;
                        tmem_st32(s_tmem + (uint32_t)(cc * 32), *reinterpret_cast<uint32_t(*)[32]>(&xa[0]));
                    }
                    tmem_st_wait();
                }
                // each chunk on its way while the one before is worked on; the last two stay for the exponentials
                load(xa, 0);
                tmem_ld_wait();
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {
                    load(xb, 2 * h + 1);
                    maximum(xa);
                    tmem_ld_wait();
                    if (h == 0) load(xa, 2);
                    maximum(xb);
                    tmem_ld_wait();
                }
                const float top = max3_nan(mx[0], mx[1], mx[1]) * args.sl2;
                // The tile before this one is of the same turn of the buffers, or (buffer 0) of the last. Its reference is
                // waited for even where it is another unit's: whoever publishes has read the one before, so that none
                // is overwritten unread. The last unit's result is drained before any wait on this unit's tiles, whose
                // first P V waits for it.
                if (j > 0 && d_lt >= 0 && !(ok = drain())) break;
                if (!(ok = warp_wait(&max_bar[prev * 4 + q], w == 0 ? phase ^ 1u : phase, abort_flag))) break;
                float mn = top;  // -inf while the row has seen nothing (or scores of -inf alone), whatever comes after
                if (j > 0) {
                    const float mp = ref_m[prev * 128 + row];
                    mn = top <= mp + kLazy ? mp : top;
                    if (__any_sync(0xFFFFFFFFu, mn != mp)) {
                        // O still holds sums relative to mp: wait for the last P V, then move it to mn
                        if (!(ok = warp_wait(&pv_done[prev], w == 0 ? phase ^ 1u : phase, abort_flag))) break;
                        tc_fence_after();
                        const float f = mn == mp ? 1.0f : ex2_ftz(mp - mn);
#pragma unroll 1
                        for (int cc = 0; cc < D / 32; ++cc) {
                            uint32_t r[32];
                            tmem_ld32(o_tmem + (uint32_t)(cc * 32), r);
                            tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * f);
                            tmem_st32(o_tmem + (uint32_t)(cc * 32), r);
                        }
                    }
                }
                ref_m[w * 128 + row] = mn;
                __syncwarp();
                if (lane == 0) mbar_arrive(&max_bar[w * 4 + q]);
                if (j >= NB && m != mn) l *= ex2_ftz(m - mn);
                m = mn;
                float2 s[2] = {both(0.0f), both(0.0f)};
                const float2 sl2 = both(args.sl2), off = both(m == -INFINITY ? 0.0f : -m);
                // a chunk's P, as the at-th 16 of the buffer's last 64 columns: the scores there are read by then
                auto probability = [&](float(&x)[32], int at) {
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float2 y = fma2(make_float2(x[2 * e], x[2 * e + 1]), sl2, off);
                        const float2 p2 = make_float2(ex2_ftz(y.x), ex2_ftz(y.y));
                        s[e & 1] = add2(s[e & 1], p2);
                        pk[e] = pack_bf16(p2.x, p2.y);
                    }
                    tmem_st16(s_tmem + (uint32_t)(64 + at * 16), pk);
                };
                // keys 64 to 127, whose scores are here, then the others read again
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {
                    probability(xa, 2 * h);
                    if (h == 0) load(xa, 0);
                    probability(xb, 2 * h + 1);
                    if (h == 0) {
                        load(xb, 1);
                        tmem_ld_wait();
                    }
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[2 * w + h]);
                }
                l += (s[0].x + s[0].y) + (s[1].x + s[1].y);
                phase ^= 1u;
                if (d_lt >= 0 && !(ok = drain())) break;
            }
            if (!ok) break;
            turn = j - nt;
            if (d_lt >= 0 && !(ok = drain())) break;  // a unit without a tile of this warpgroup
            fin[(lt & 1) * (NB * 128) + w * 128 + row] = make_float2(m, l);
            __syncwarp();
            if (lane == 0) mbar_arrive(&fin_bar[(lt & 1) * 4 + q]);
            d_lt = lt, d_nt = nt, d_h = un.h, d_shift = shift;
            d_tok = (int64_t)un.tok0 + row - shift;
            // the last tile's buffer: this warpgroup's next tile is `turn` tiles into the next unit
            d_last = w - turn - 1;
            if (d_last < 0) d_last += NB;
        }
        if (ok && d_lt >= 0) ok = drain();
        if (!ok) *abort_flag = 1;
    }

    tc_fence_before();
    __syncthreads();
    settle(abort_flag);
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// The tokens of the batch's last block, 128 when it is full.
int tail_tokens(const R97bPacked& p) {
    for (int b = p.n_blocks - 1; b >= 0; --b) {  // (short sequences stand last)
        const int32_t* e = p.k_blocks_host + 4 * (int64_t)b;
        if ((int64_t)e[0] + e[1] == p.T) return (e[1] - 1) % kBlk + 1;
    }
    return 0;
}
// An operand's maps: the batch's, and the last block's (the first again where that is full).
bool make_maps(CUtensorMap* m, const R97bHeadRows& r, int64_t heads, int32_t D, int64_t T, int tail, int box_rows) {
    if (!make_rows_map(&m[0], r, heads, D, T, kBlk, box_rows)) return false;
    m[1] = m[0];
    return tail == 0 || tail == kBlk || make_rows_map(&m[1], r, heads, D, T, tail, box_rows);
}

template <int D>
int launch_fwd(const R97bPacked& p, const R97bAttnPackedFwd& a, cudaStream_t st) {
    using C = FCfg<D>;
    static_assert(C::kSmemBytes <= 232448, "shared memory");
    const int tail = tail_tokens(p);
    CUtensorMap q[2], k[2], v[2];
    if (!make_maps(q, a.q, a.Hq, D, p.T, tail, kBlk) || !make_maps(k, a.k, a.Hkv, D, p.T, tail, kBlk) ||
        !make_maps(v, a.v, a.Hkv, D, p.T, tail, C::kVRows))
        return R97B_EINVAL;
    FwdArgs r{};
    r.tail_n = tail;
    r.blocks = reinterpret_cast<const int4*>(p.q_blocks);
    r.o = reinterpret_cast<__nv_bfloat16*>(a.o.ptr);
    r.lse = a.lse;
    r.o_tok = a.o.tok, r.o_head = a.o.head, r.ld_lse = a.ld_lse;
    r.Hq = a.Hq, r.grp = a.Hq / a.Hkv;
    r.T = (int32_t)p.T;
    r.q_head = (int32_t)a.q.head, r.k_head = (int32_t)a.k.head, r.v_head = (int32_t)a.v.head;
    r.q = reinterpret_cast<const __nv_bfloat16*>(a.q.ptr), r.q_tok = a.q.tok;
    r.k = reinterpret_cast<const __nv_bfloat16*>(a.k.ptr), r.k_tok = a.k.tok;
    r.v = reinterpret_cast<const __nv_bfloat16*>(a.v.ptr), r.v_tok = a.v.tok;
    r.sl2 = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * kLog2e;
    r.sign = a.scale == 0.0f ? 0.0f : (a.scale < 0.0f ? -1.0f : 1.0f);
    if (!smem_opt_in(fwd_kernel<D>, C::kSmemBytes)) return R97B_ELAUNCH;
    fwd_kernel<D><<<p.n_blocks * a.Hq, C::kThreads, C::kSmemBytes, st>>>(q[0], k[0], v[0], q[1], k[1], v[1], r);
    return launch_status();
}

// ------------------------------------------------------------------------------------------ backward

// The tiles of the backward, recomputed from q, k and the forward's lse. Four kinds of pass share one kernel; each
// keeps its accumulators in TMEM over a unit's tiles and writes every result once, in a fixed order (no atomics):
//
//   kDQ   rows = queries: S = Q K^T, dP = dO V^T, dS = P o (dP - delta);        dQ += dS K
//   kDKV  rows = keys:    S^T = K Q^T, dP^T = V dO^T;   dV += P^T dO and dK += dS^T Q     (D = 128)
//   kDV   rows = keys:    S^T = K Q^T;                  dV += P^T dO                      (D = 256)
//   kDK   rows = keys:    S^T = K Q^T, dP^T = V dO^T;   dK += dS^T Q                      (D = 256)
//
// At D = 256 dV and dK of 128 keys fill the 512 TMEM columns by themselves, so they are two passes, the second computing
// S^T again. The rows' operands stay in shared memory for the unit; the others stream through a ring of 16 KB chunks,
// K-major for the score products and MN-major for the accumulating ones, whose A operand (P or dS, bf16) the
// elementwise threads write over their own columns of the scores' TMEM. Each thread owns a row and each of the four
// warpgroups 32 of its columns; the next tile's S is issued before the accumulating products, so its exponentials run
// beside them, and only dS (a product and a rounding) stands between dP and the products that read it.
// kDQ goes first and leaves every row's delta = dO . O for the others: it has dO in shared memory. (A kernel of its own,
// bound by its reads of o and dout, cost more: a chat batch of 16384 tokens, 8/2 heads of 128, 72 us for the two, 66 in one;
// 8192 tokens of 16/4 heads of 256, 149 and 134, then.) At D = 128 both of a column block's products read one 32 KB copy of it:
// 12301 tokens 1.68 -> 1.55 ms.
enum Kind { kDQ = 0, kDKV = 1, kDV = 2, kDK = 3 };

constexpr int kThreads = 640;  // warps 0, 3: TMA, warp 1: MMA, warp 2: the columns' statistics; four warpgroups after
constexpr int kSoftWarps = 16;
constexpr int kCtrlRegs = 64, kSoftRegs = 104;  // 128 x 64 + 512 x 104 = 640 x 96, what the launch holds
static_assert(128 * kCtrlRegs + 512 * kSoftRegs <= 640 * 96, "register split");

template <int D, int KIND>
struct BCfg {
    static constexpr bool kDP = KIND != kDV;          // needs dP (a second resident operand, delta)
    static constexpr bool kKeys = KIND != kDQ;        // rows are keys: lse and delta run along the columns
    static constexpr int kABytes = kBlk * D * 2;
    // At D = 128 the ring holds whole column blocks of 32 KB, each read by both of its products (K-major for the scores,
    // MN-major for the accumulating one); at 256 it holds 16 KB chunks, loaded once for either.
    static constexpr bool kWhole = D == 128;
    static constexpr int kSlot = kWhole ? kABytes : kChunk;
    static constexpr int kStages = kWhole ? 5 : (kDP ? 6 : 9);
    static constexpr int kRingOff = (kDP ? 2 : 1) * kABytes;
    static constexpr int kBarOff = kRingOff + kStages * kSlot;
    static constexpr int kStatOff = kBarOff + 640;    // kKeys: float [2 (stage)][-lse log2 e, -delta][128]
    static constexpr int kSmemBytes = kStatOff + 2048;  // kDQ: float [4][128], a row's P o dP by column quarter
    static constexpr int kVRows = kChunk / (D * 2);
};

struct TailMaps {
    CUtensorMap a0, a1, b0, b1, c0;
};
struct BwdArgs {
    const int4* blocks;
    const float* lse;
    float* delta;                      // written by kDQ, read by the others, which follow it
    int64_t ld_lse, ld_delta;
    const __nv_bfloat16* o;            // kDQ: the forward's output
    int64_t o_tok, o_head;
    __nv_bfloat16 *out0, *out1;        // kDQ: dq; kDKV: dv, dk; kDV: dv; kDK: dk
    int64_t tok0, head0, tok1, head1;
    int32_t a0_head, a1_head, b0_head, b1_head, c0_head;
    int32_t T, tail_n;                 // tokens of the batch, and of its last block
    const __nv_bfloat16 *a0, *a1, *b0, *b1, *c0;  // the operands again, for copy_chunk
    int64_t a0_tok, a1_tok, b0_tok, b1_tok, c0_tok;
    int32_t heads, grp;                // the rows' heads (query heads for kDQ, key/value heads else)
    // keys: the first split_blocks blocks' query heads go to `parts` units each, launched behind the first_blocks
    // blocks after them (whose whole units are longer)
    int32_t split_blocks, parts, first_blocks;
    float *part0, *part1;              // and their sums, f32 [split block][head][part] x part_at, here
    float sl2, scale;
};

// Where a unit's f32 sums of four columns (the cg-th four of row `row`) stand, in float4: the rows of a column group are
// neighbours, as the threads that write and read them are (row by row, a unit's stores took 4.5 us at D = 256).
template <int D>
__device__ __forceinline__ int64_t part_at(int64_t slot, int cg, int row) {
    return (slot * (D / 4) + cg) * kBlk + row;
}

// A unit's tiles: kDQ walks the key blocks up to its own; the others every query block from their own on, head by head.
template <int KIND>
struct Walk {
    int h, i, n, seq0, tok0, len, m, tiles, head0;
    int slot;  // the unit's partial sums, or -1 when it writes its rows' results
    __device__ Walk(const BwdArgs& a, int u) {
        int b, part = 0, heads = KIND == kDQ ? 1 : a.grp;  // the tiles' query heads
        slot = -1;
        if (KIND != kDQ) u -= a.first_blocks * a.heads;
        if (KIND != kDQ && u >= 0 && u < a.split_blocks * a.heads * a.parts) {
            slot = u;
            b = u / (a.heads * a.parts);
            h = (u - b * a.heads * a.parts) / a.parts;
            part = u % a.parts;
            heads /= a.parts;
        } else {
            if (KIND != kDQ) {  // before the split ones, or behind them
                u += a.first_blocks * a.heads;
                u += u < a.first_blocks * a.heads ? a.split_blocks * a.heads : -a.split_blocks * a.heads * (a.parts - 1);
            }
            b = u / a.heads;
            h = u - b * a.heads;
        }
        const int4 e = a.blocks[b];
        head0 = KIND == kDQ ? h / a.grp : h * a.grp + part * heads;
        i = e.z;
        seq0 = e.x;
        len = e.y;
        tok0 = seq0 + i * kBlk;
        n = min(kBlk, len - i * kBlk);
        m = KIND == kDQ ? i + 1 : (len + kBlk - 1) / kBlk - i;
        tiles = m * heads;
    }
    __device__ int shift() const { return kBlk - n; }
    // the first tile's column block and head, and the step to the next one's
    __device__ int first_block() const { return KIND == kDQ ? 0 : i; }
    __device__ int first_head() const { return head0; }
    __device__ void step(int& blk, int& head) const {
        if (++blk == i + m && KIND != kDQ) {
            blk = i;
            ++head;
        }
    }
    __device__ int shift_of(int blk) const { return kBlk - min(kBlk, len - blk * kBlk); }
};

template <int D, int KIND>
__global__ void __launch_bounds__(kThreads, 1)
    bwd_kernel(const __grid_constant__ CUtensorMap tA0, const __grid_constant__ CUtensorMap tA1,
               const __grid_constant__ CUtensorMap tB0, const __grid_constant__ CUtensorMap tB1,
               const __grid_constant__ CUtensorMap tC0, const __grid_constant__ TailMaps tails, const BwdArgs args) {
    using C = BCfg<D, KIND>;
    constexpr int ND = D / 64;
    constexpr int kVC = kBlk / C::kVRows;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* ring = smem + C::kRingOff;
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
    const UnitQueue queue{reinterpret_cast<uint4*>(full_bar), full_bar + 8, full_bar + 12,
                          reinterpret_cast<volatile int*>(full_bar + 16)};
    volatile int* abort_flag = queue.abort;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(full_bar + 16) + 1;
    full_bar += 17;
    uint64_t* empty_bar = full_bar + C::kStages;
    uint64_t* a_full = empty_bar + C::kStages;   // [2]
    uint64_t* a_empty = a_full + 2;              // [2]
    uint64_t* s_full = a_empty + 2;              // [2]
    uint64_t* s_free = s_full + 2;               // all but kDV: S read into registers
    uint64_t* p_full = s_free + 1;               // [2] kDV: P written
    uint64_t* dp_full = p_full + 2;
    uint64_t* ds_full = dp_full + 1;
    uint64_t* acc_full = ds_full + 1;
    uint64_t* acc_empty = acc_full + 1;
    uint64_t* stat_full = acc_empty + 1;         // [2]
    uint64_t* stat_empty = stat_full + 2;        // [2]
    uint64_t* sum_bar = stat_empty + 2;          // [4] kDQ: a lane quarter's row sums written
    float* stats = reinterpret_cast<float*>(smem + C::kStatOff);

    const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0);
    const int lane = threadIdx.x & 31;
    if (smem_u32(smem) & 1023u) {  // the swizzled tiles need it; the attribute above asks for it
        if (threadIdx.x == 0) atomicOr(&g_device_error, kErrArgs);
        return;
    }
    if (threadIdx.x == 0) {
        queue.init(4 + kSoftWarps);
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&a_full[b], 1);
            mbar_init(&a_empty[b], 1);
            mbar_init(&s_full[b], 1);
            mbar_init(&p_full[b], kSoftWarps);
            mbar_init(&stat_full[b], 1);
            mbar_init(&stat_empty[b], kSoftWarps);
        }
        for (int b = 0; b < 4; ++b) mbar_init(&sum_bar[b], 4);
        mbar_init(s_free, kSoftWarps);
        mbar_init(dp_full, 1);
        mbar_init(ds_full, kSoftWarps);
        mbar_init(acc_full, 1);
        mbar_init(acc_empty, kSoftWarps);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch(&tA0);
        tma_prefetch(&tB0);
        tma_prefetch(&tC0);
        if (C::kDP) {
            tma_prefetch(&tA1);
            tma_prefetch(&tB1);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_slot, 0);
    const uint32_t acc0 = tmem + 256u, acc1 = tmem + 384u;  // acc1: kDKV's dK

    if (warp < 4) {
        set_max_regs_dec<kCtrlRegs>();
        if (warp == 0 || warp == 3) {
            // --------------------------------------------------------- TMA producers: every other chunk each
            const uint32_t lead = elect_one();
            const int p = warp == 3;
            int stage = p;
            uint32_t phase = 0;
            bool ok = true;
            for (int u = blockIdx.x, lt = 0; ok && u >= 0; u = ok ? queue.next(lt) : -1, ++lt) {
                const Walk<KIND> wk(args, u);
                if (p == 0 || C::kDP) {  // a resident operand each
                    if (!(ok = warp_wait(&a_empty[p], (uint32_t)(lt & 1) ^ 1u, abort_flag))) break;
                    const int x = wk.h * (p ? args.a1_head : args.a0_head), at = map_of(wk.tok0, wk.n, args.T, args.tail_n);
                    if (at < 0) {
                        const int64_t step = p ? args.a1_tok : args.a0_tok;
#pragma unroll 1
                        for (int s = 0; s < ND; ++s)
                            copy_chunk(smem + p * C::kABytes + s * kChunk, (p ? args.a1 : args.a0) + wk.tok0 * step + x + 64 * s,
                                       step, 7, 0, wk.shift());
                        copies_done(&a_full[p], lead);
                    } else if (lead) {
                        const CUtensorMap* map = p ? (at ? &tails.a1 : &tA1) : (at ? &tails.a0 : &tA0);
                        mbar_expect_tx(&a_full[p], C::kABytes);
                        for (int s = 0; s < ND; ++s)
                            tma_load_3d(smem + p * C::kABytes + s * kChunk, map, &a_full[p], x + 64 * s, -wk.shift(), wk.tok0);
                    }
                }
                int blk0 = 0, head0 = 0, blk1 = wk.first_block(), head1 = wk.first_head();  // of tiles j and j + 1
                if constexpr (C::kWhole) {
                    // each of the two warps its operand's blocks, in slots taken in turn
                    const int head_stride = p ? args.b1_head : args.b0_head;
                    for (int j = 0; j < wk.tiles && ok; ++j) {
                        if (p && j + 1 == wk.tiles && !(ok = queue.ask(lt, lead))) break;
                        if (!(ok = warp_wait(&empty_bar[stage], phase ^ 1u, abort_flag))) break;
                        const int tok = wk.seq0 + blk1 * kBlk, shift = wk.shift_of(blk1), x = head1 * head_stride;
                        const int at = map_of(tok, kBlk - shift, args.T, args.tail_n);
                        if (at < 0) {
                            const int64_t step = p ? args.b1_tok : args.b0_tok;
#pragma unroll 1
                            for (int ch = 0; ch < ND; ++ch)
                                copy_chunk(ring + stage * C::kSlot + ch * kChunk, (p ? args.b1 : args.b0) + tok * step + x + 64 * ch,
                                           step, 7, 0, shift);
                            copies_done(&full_bar[stage], lead);
                        } else if (lead) {
                            const CUtensorMap* map = p ? (at ? &tails.b1 : &tB1) : (at ? &tails.b0 : &tB0);
                            mbar_expect_tx(&full_bar[stage], C::kSlot);
#pragma unroll
                            for (int ch = 0; ch < ND; ++ch)
                                tma_load_3d(ring + stage * C::kSlot + ch * kChunk, map, &full_bar[stage], x + 64 * ch, -shift, tok);
                        }
                        if ((stage += 2) >= C::kStages) {
                            stage -= C::kStages;
                            phase ^= 1u;
                        }
                        wk.step(blk1, head1);
                    }
                } else {
                    // a step's streams, in the order the products take them: the next tile's column block for S (K-major), this
                    // tile's for the accumulating product (MN-major), the next tile's for dP. Rolled: the warps share an
                    // instruction cache that unrolled copies do not fit in beside the softmax.
#pragma unroll 1
                    for (int j = -1; j < wk.tiles && ok; ++j) {
                        if (p && j + 1 == wk.tiles && !(ok = queue.ask(lt, lead))) break;
#pragma unroll 1
                        for (int s = 0; s < 3 && ok; ++s) {
                            const bool mn = s == 1;
                            const int tile = mn ? j : j + 1;
                            if (tile < 0 || tile >= wk.tiles || (s == 2 && !C::kDP)) continue;
                            const int head_stride = s == 0 ? args.b0_head : (s == 1 ? args.c0_head : args.b1_head);
                            const int blk = mn ? blk0 : blk1, x = (mn ? head0 : head1) * head_stride;
                            const int r0 = -wk.shift_of(blk), tok = wk.seq0 + blk * kBlk;
                            const int at = map_of(tok, kBlk + r0, args.T, args.tail_n);
                            const CUtensorMap* map = at == 1 ? (s == 0 ? &tails.b0 : (s == 1 ? &tails.c0 : &tails.b1))
                                                             : (s == 0 ? &tB0 : (s == 1 ? &tC0 : &tB1));
#pragma unroll 1
                            for (int ch = p; ch < (mn ? kVC : ND); ch += 2) {
                                if (!(ok = warp_wait(&empty_bar[stage], phase ^ 1u, abort_flag))) break;
                                uint8_t* st = ring + stage * kChunk;
                                if (at < 0) {
                                    const int64_t step = s == 0 ? args.b0_tok : (s == 1 ? args.c0_tok : args.b1_tok);
                                    const __nv_bfloat16* rows = s == 0 ? args.b0 : (s == 1 ? args.c0 : args.b1);
                                    copy_chunk(st, rows + tok * step + x + (mn ? 0 : 64 * ch), step, mn ? (C::kVRows == 64 ? 6 : 5) : 7,
                                               mn ? ch * C::kVRows : 0, -r0);
                                    copies_done(&full_bar[stage], lead);
                                } else if (lead) {
                                    mbar_expect_tx(&full_bar[stage], kChunk);
                                    if (mn) {
#pragma unroll
                                        for (int n = 0; n < ND; ++n)
                                            tma_load_3d(st + n * (C::kVRows * 128), map, &full_bar[stage], x + 64 * n,
                                                        ch * C::kVRows + r0, tok);
                                    } else {
                                        tma_load_3d(st, map, &full_bar[stage], x + 64 * ch, r0, tok);
                                    }
                                }
                                if ((stage += 2) >= C::kStages) {
                                    stage -= C::kStages;
                                    phase ^= 1u;
                                }
                            }
                        }
                        blk0 = blk1, head0 = head1;
                        wk.step(blk1, head1);
                    }
                }
            }
        } else if (warp == 1) {
            const uint32_t lead = elect_one();
            // --------------------------------------------------------- MMA issuer
            constexpr uint32_t idesc_s = make_idesc_bf16(kBlk, kBlk, 0, 0);
            constexpr uint32_t idesc_c = make_idesc_bf16(kBlk, D, 0, 1);
            int stage = 0, g = 0;  // g: the current unit's first tile
            uint32_t phase = 0;
            bool ok = true;
            const uint32_t a_lo = sdesc_lo(smem_u32(smem), 16);
            const uint32_t b_lo = sdesc_lo(smem_u32(ring), 16);
            const uint32_t c_lo = sdesc_lo(smem_u32(ring), C::kWhole ? kChunk : C::kVRows * 128);
            auto chunk = [&]() -> bool {  // the next ring chunk is there
                ok = ok && warp_wait(&full_bar[stage], phase, abort_flag);
                tc_fence_after();
                return ok;
            };
            auto next = [&]() {
                umma_commit_by(lead, &empty_bar[stage]);
                if (++stage == C::kStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            };
            // kWhole: the tile's operand `which` (0, 1) is in slot (2 tile + which) % kStages
            auto score = [&](int resident, uint32_t d) {
                if constexpr (C::kWhole) {
                    ok = ok && warp_wait(&full_bar[stage], phase, abort_flag);
                    tc_fence_after();
                    if (!ok) return;
#pragma unroll
                    for (int kb = 0; kb < ND; ++kb) {
                        const uint32_t a = a_lo + (uint32_t)(resident * (C::kABytes >> 4) + kb * kChunkLo);
                        const uint32_t b = b_lo + (uint32_t)(stage * (C::kSlot >> 4) + kb * kChunkLo);
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            umma_f16_by(lead, d, sdesc(a + kk * 2, kDescHi), sdesc(b + kk * 2, kDescHi), idesc_s,
                                        (kb > 0 || kk > 0) ? 1u : 0u);
                    }
                    if (KIND == kDQ && resident == 1) umma_commit_by(lead, &empty_bar[stage]);  // V is not read again
                    if (++stage == C::kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                } else {
#pragma unroll 1
                    for (int kb = 0; kb < ND; ++kb) {
                        if (!chunk()) return;
                        const uint32_t a = a_lo + (uint32_t)(resident * (C::kABytes >> 4) + kb * kChunkLo);
                        const uint32_t b = b_lo + (uint32_t)(stage * kChunkLo);
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            umma_f16_by(lead, d, sdesc(a + kk * 2, kDescHi), sdesc(b + kk * 2, kDescHi), idesc_s,
                                        (kb > 0 || kk > 0) ? 1u : 0u);
                        next();
                    }
                }
            };
            // d (+)= a x the tile's operand `which`, MN-major
            int held = 0;  // kWhole: the slot of the tile's operand 0
            auto accumulate = [&](uint32_t a, uint32_t d, bool first, int which) {
                if constexpr (C::kWhole) {
                    int at = held + which;
                    if (at >= C::kStages) at -= C::kStages;
                    const uint32_t b = c_lo + (uint32_t)(at * (C::kSlot >> 4));
#pragma unroll
                    for (int k16 = 0; k16 < kBlk / 16; ++k16)
                        umma_f16_ts_by(lead, d, a + (uint32_t)quarter_col(k16), sdesc(b + k16 * 128, kDescHi), idesc_c,
                                       (!first || k16 > 0) ? 1u : 0u);
                    umma_commit_by(lead, &empty_bar[at]);
                } else {
#pragma unroll 1
                    for (int ch = 0; ch < kVC; ++ch) {
                        if (!chunk()) return;
                        const uint32_t b = c_lo + (uint32_t)(stage * kChunkLo);
#pragma unroll
                        for (int kk = 0; kk < C::kVRows / 16; ++kk) {
                            umma_f16_ts_by(lead, d, a + (uint32_t)quarter_col(ch * (C::kVRows / 16) + kk),
                                           sdesc(b + kk * 128, kDescHi), idesc_c, (!first || ch > 0 || kk > 0) ? 1u : 0u);
                        }
                        next();
                    }
                }
            };
            auto wait = [&](uint64_t* bar, int n) {  // the bar's n-th completion
                ok = ok && warp_wait(bar, (uint32_t)(n & 1), abort_flag);
                tc_fence_after();
            };
            for (int u = blockIdx.x, lt = 0; ok && u >= 0; u = ok ? queue.next(lt) : -1, ++lt) {
                const Walk<KIND> wk(args, u);
                const int n = wk.tiles;
                auto issue_s = [&](int j) {
                    const int gj = g + j, b = KIND == kDV ? (gj & 1) : 0;
                    if (KIND != kDV && gj > 0) wait(s_free, gj - 1);
                    if (j == 0) wait(&a_full[0], lt);
                    if (!ok) return;
                    score(0, tmem + (uint32_t)(b * kBlk));
                    umma_commit_by(lead, &s_full[b]);
                    if (j + 1 == n) umma_commit_by(lead, &a_empty[0]);
                };
                auto issue_dp = [&](int j) {
                    if (j == 0) wait(&a_full[1], lt);
                    if (!ok) return;
                    score(1, tmem + (uint32_t)kBlk);
                    umma_commit_by(lead, dp_full);
                    if (j + 1 == n) umma_commit_by(lead, &a_empty[1]);
                };
                issue_s(0);
                if (C::kDP) issue_dp(0);
                for (int j = 0; j < n && ok; ++j) {
                    const int gj = g + j, b = KIND == kDV ? (gj & 1) : 0;
                    const bool more = j + 1 < n;
                    if (more) issue_s(j + 1);
                    if (KIND == kDV)
                        wait(&p_full[b], gj >> 1);
                    else
                        wait(ds_full, gj);
                    if (j == 0) wait(acc_empty, lt + 1);
                    if (!ok) break;
                    accumulate(tmem + (uint32_t)(KIND == kDV ? b * kBlk : kBlk), acc0, j == 0, KIND == kDKV ? 1 : 0);
                    if (KIND == kDKV) accumulate(tmem + (uint32_t)(kBlk + 16), acc1, j == 0, 0);
                    if ((held += 2) >= C::kStages) held -= C::kStages;
                    if (more && C::kDP) issue_dp(j + 1);
                }
                if (!ok) break;
                umma_commit_by(lead, acc_full);
                g += n;
            }
        } else if (KIND == kDQ) {
            // --------------------------------------------------------- the next unit's output rows, into L2 for delta
            for (int u = blockIdx.x, lt = 0; u >= 0; u = queue.next(lt), ++lt) {
                const Walk<KIND> wk(args, u);
                if (wk.tiles == 1) continue;
                const __nv_bfloat16* op = args.o + (int64_t)wk.tok0 * args.o_tok + wk.h * args.o_head;
                for (int k = lane; k < wk.n * (D / 64); k += 32)
                    prefetch_l2(op + k / (D / 64) * args.o_tok + k % (D / 64) * 64);
            }
        } else {
            // --------------------------------------------------------- the columns' lse and delta, a tile ahead
            int g = 0;
            bool ok = true;
            for (int u = blockIdx.x, lt = 0; ok && u >= 0; u = ok ? queue.next(lt) : -1, ++lt) {
                const Walk<KIND> wk(args, u);
                int blk = wk.first_block(), h = wk.first_head();
                for (int j = 0; j < wk.tiles; ++j, ++g, wk.step(blk, h)) {
                    const int shift = wk.shift_of(blk), st = g & 1;
                    const int64_t tok = (int64_t)wk.seq0 + blk * kBlk - shift;
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int col = e * 32 + lane;
                        // negated, for the sums that take them; a column before the block's first token: 2^-inf = 0
                        v[e] = col >= shift ? args.lse[h * args.ld_lse + tok + col] * -kLog2e : -INFINITY;
                        v[4 + e] = C::kDP && col >= shift ? -args.delta[h * args.ld_delta + tok + col] : 0.0f;
                    }
                    if (!(ok = warp_wait(&stat_empty[st], (uint32_t)((g >> 1) & 1) ^ 1u, abort_flag))) break;
                    float* s = stats + st * 256;
#pragma unroll
                    for (int e = 0; e < 8; ++e) s[e * 32 + lane] = v[e];
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&stat_full[st]);
                }
            }
        }
    } else {
        // ------------------------------------------------------------- probabilities, dS, and the results' rows
        set_max_regs_inc<kSoftRegs>();
        const int q = warp & 3, w = (warp - 4) >> 2;
        const int row = q * 32 + lane;
        const uint32_t lane_off = (uint32_t)(q * 32) << 16;
        const uint32_t mine = tmem + lane_off + (uint32_t)(w * 32);  // this thread's columns of S (and, 128 on, of dP)
        int g = 0;
        uint32_t sum_phase = 0;
        bool ok = true;
        // the unit whose result is still in TMEM: its number, head, first valid row, partial slot, and this row's token
        int d_lt = -1, d_h = 0, d_shift = 0, d_slot = -1;
        int64_t d_tok = 0;
        auto drain = [&]() -> bool {
            if (!warp_wait(acc_full, (uint32_t)(d_lt & 1), abort_flag)) return false;
            tc_fence_after();
#pragma unroll
            for (int r = 0; r < (KIND == kDKV ? 2 : 1); ++r) {
                // dV takes no scale; dS is kept unscaled in bf16, so dQ and dK take it here
                const float f = (KIND == kDV || (KIND == kDKV && r == 0)) ? 1.0f : args.scale;
                const int64_t tok = r ? args.tok1 : args.tok0;
                __nv_bfloat16* op = r ? args.out1 + d_tok * args.tok1 + d_h * args.head1
                                      : args.out0 + d_tok * args.tok0 + d_h * args.head0;
                const uint32_t src = (r ? acc1 : acc0) + lane_off + (uint32_t)(w * (D / 4));
#pragma unroll 1
                for (int cc = 0; cc < D / 128; ++cc) {
                    uint32_t v[32];
                    __syncwarp();
                    tmem_ld32(src + (uint32_t)(cc * 32), v);
                    tmem_ld_wait();
                    if (C::kKeys && d_slot >= 0) {
                        if (row < d_shift) continue;
                        float4* pp = reinterpret_cast<float4*>(r ? args.part1 : args.part0) +
                                     part_at<D>(d_slot, w * (D / 16) + cc * 8, row);
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            pp[k * kBlk] = make_float4(__uint_as_float(v[4 * k]), __uint_as_float(v[4 * k + 1]),
                                                __uint_as_float(v[4 * k + 2]), __uint_as_float(v[4 * k + 3]));
                    } else {
                        store_rows32(op + w * (D / 4) + cc * 32, tok, row, d_shift, v, f);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty);
            d_lt = -1;
            return true;
        };
        for (int u = blockIdx.x, lt = 0; ok && u >= 0; u = ok ? queue.next(lt) : -1, ++lt) {
            const Walk<KIND> wk(args, u);
            const int shift = wk.shift();
            const int64_t tok = (int64_t)wk.tok0 + row - shift;
            float lse2 = 0.0f, delta = 0.0f;
            if (!C::kKeys && row >= shift) lse2 = args.lse[wk.h * args.ld_lse + tok] * kLog2e;
            if (!C::kKeys && wk.tiles > 1) {
                // delta = dO . O, this warp's quarter of its rows, while the tensor core has the first scores to go on with:
                // kLanes lanes a row, so that a load touches whole lines. dO is in shared memory until the unit's last
                // dP, which waits for this warp's first dS.
                constexpr int kLanes = D / 32, kRows = 32 / kLanes;  // kRows rows a step, kLanes steps
                const int at = w * kLanes + lane % kLanes;           // the lane's 16-byte piece of a row
                const __nv_bfloat16* op = args.o + wk.h * args.o_head + at * 8;
                uint4 o[kLanes];
#pragma unroll
                for (int c = 0; c < kLanes; ++c) {
                    const int r = q * 32 + c * kRows + lane / kLanes - shift;
                    o[c] = r >= 0 ? *reinterpret_cast<const uint4*>(op + ((int64_t)wk.tok0 + r) * args.o_tok)
                                  : make_uint4(0, 0, 0, 0);
                }
                if (!(ok = warp_wait(&a_full[1], (uint32_t)(lt & 1), abort_flag))) break;
                float part[kLanes];
#pragma unroll
                for (int c = 0; c < kLanes; ++c) {
                    const int r = q * 32 + c * kRows + lane / kLanes;
                    const uint4 g4 = *reinterpret_cast<const uint4*>(smem + C::kABytes + (at >> 3) * kChunk + r * 128 +
                                                                     (((at & 7) ^ (r & 7)) << 4));  // 128-byte swizzle
                    const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(&o[c]);
                    const __nv_bfloat162* y = reinterpret_cast<const __nv_bfloat162*>(&g4);
                    part[c] = 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 xf = __bfloat1622float2(x[e]), yf = __bfloat1622float2(y[e]);
                        part[c] = fmaf(xf.x, yf.x, part[c]);
                        part[c] = fmaf(xf.y, yf.y, part[c]);
                    }
                }
                // the lanes of a row sum its pieces, each ending with another step's row; then row `lane` to each lane
#pragma unroll
                for (int half = kLanes / 2; half > 0; half >>= 1) {
                    const bool upper = lane & half;
#pragma unroll
                    for (int c = 0; c < half; ++c) {
                        const float give = upper ? part[c] : part[c + half];
                        part[c] = (upper ? part[c + half] : part[c]) + __shfl_xor_sync(0xFFFFFFFFu, give, half);
                    }
                }
                delta = __shfl_sync(0xFFFFFFFFu, part[0], lane % kRows * kLanes + lane / kRows);
            }
            for (int j = 0, jm = 0; j < wk.tiles; ++j, ++g) {
                const int b = KIND == kDV ? (g & 1) : 0;
                // the diagonal tile: the last of kDQ, the first of each query head else
                const bool diag = C::kKeys ? jm == 0 : j + 1 == wk.tiles;
                if (++jm == wk.m) jm = 0;
                const float* st = stats + (g & 1) * 256 + w * 32;
                if (C::kKeys && !(ok = warp_wait(&stat_full[g & 1], (uint32_t)((g >> 1) & 1), abort_flag))) break;
                if (!(ok = warp_wait(&s_full[b], (uint32_t)((KIND == kDV ? g >> 1 : g) & 1), abort_flag))) break;
                tc_fence_after();
                float p[32];
                tmem_ld32(mine + (uint32_t)(b * kBlk), *reinterpret_cast<uint32_t(*)[32]>(&p[0]));
                tmem_ld_wait();
                if (KIND != kDV) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(s_free);
                }
                const float2 sl2 = both(args.sl2);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float2 y = make_float2(p[2 * e], p[2 * e + 1]);
                    if (C::kKeys) {  // the column's -lse
                        y = fma2(y, sl2, *reinterpret_cast<const float2*>(st + 2 * e));
                    } else {
                        y = fma2(y, sl2, both(-lse2));
                    }
                    p[2 * e] = ex2_ftz(y.x);
                    p[2 * e + 1] = ex2_ftz(y.y);
                }
                // on the diagonal only the warp's own 32 columns are seen in part, those on one side not at all
                if (diag && (C::kKeys ? w <= q : (w >= q || w * 32 < shift))) {
                    const int at = row - w * 32, lo = shift - w * 32;
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (C::kKeys ? e < at : (e > at || e < lo)) p[e] = 0.0f;
                }
                uint32_t pk[16];
                if (KIND == kDV || KIND == kDKV) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) pk[e] = pack_bf16(p[2 * e], p[2 * e + 1]);
                }
                if (KIND == kDV) {
                    tmem_st16(mine + (uint32_t)(b * kBlk), pk);
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[b]);
                } else {
                    if (!(ok = warp_wait(dp_full, (uint32_t)(g & 1), abort_flag))) break;
                    tc_fence_after();
                    float d[32];
                    tmem_ld32(mine + (uint32_t)kBlk, *reinterpret_cast<uint32_t(*)[32]>(&d[0]));
                    tmem_ld_wait();
                    if (KIND == kDKV) tmem_st16(mine + (uint32_t)kBlk, pk);  // P beside dS, over dP
                    if (KIND == kDQ && j == 0) {
                        // A sequence's first rows are all here, and delta is the row's sum of P o dP, in f32. With few
                        // keys dP - delta cancels, and the bf16 rounding of o in sum dO o O would cost dq and dk a
                        // quarter more error than the rounding of dS does (every later row averages it away).
                        if (wk.tiles == 1) {
#pragma unroll
                            for (int e = 0; e < 32; ++e) delta += p[e] != 0.0f ? p[e] * d[e] : 0.0f;
                        }
                        // The quarters' sums. Those of the unit before have been read: its last dS was complete before
                        // this dP was issued.
                        stats[w * kBlk + row] = delta;
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sum_bar[q]);
                        if (!(ok = warp_wait(&sum_bar[q], sum_phase, abort_flag))) break;
                        sum_phase ^= 1u;
                        delta = (stats[row] + stats[kBlk + row]) + (stats[2 * kBlk + row] + stats[3 * kBlk + row]);
                        // for the passes over the keys, which follow
                        if (w == 0 && row >= shift) args.delta[wk.h * args.ld_delta + tok] = delta;
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        float2 n = both(-delta);  // minus the row's delta, or the columns'
                        if (C::kKeys) n = *reinterpret_cast<const float2*>(st + 128 + 2 * e);
                        const float2 y = mul2(make_float2(p[2 * e], p[2 * e + 1]), add2(make_float2(d[2 * e], d[2 * e + 1]), n));
                        pk[e] = pack_bf16(y.x, y.y);
                    }
                    tmem_st16(mine + (uint32_t)(kBlk + (KIND == kDKV ? 16 : 0)), pk);
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(ds_full);
                }
                if (C::kKeys && lane == 0) mbar_arrive(&stat_empty[g & 1]);
                // the last unit's result, now that the tensor core has this unit's first products to go on with
                if (d_lt >= 0 && !(ok = drain())) break;
            }
            if (!ok) break;
            d_lt = lt, d_h = wk.h, d_shift = shift, d_slot = wk.slot, d_tok = tok;
        }
        if (ok && d_lt >= 0) ok = drain();
        if (!ok) *abort_flag = 1;
    }

    tc_fence_before();
    __syncthreads();
    settle(abort_flag);
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

int64_t delta_ld(int64_t T) { return (T + 63) / 64 * 64; }

// dk, dv rows of the split blocks: their parts summed in order. A thread sums 8 columns of a row, a warp those of 32 rows.
struct SumArgs {
    const int4* blocks;
    const float *dv_parts, *dk_parts;
    R97bHeadRows dv, dk;
    float scale;
    int32_t heads, parts;
};
template <int D>
__global__ void __launch_bounds__(256) sum_parts_kernel(const SumArgs a) {
    constexpr int kPer = 2 * kBlk * (D / 8) / 256;  // thread blocks a unit
    const int unit = (int)(blockIdx.x / kPer), at = (int)(blockIdx.x % kPer) * 256 + threadIdx.x;
    const int row = at % kBlk, c8 = at / kBlk % (D / 8), is_dk = at / (kBlk * (D / 8));
    const int b = unit / a.heads, h = unit - b * a.heads;
    const int4 e = a.blocks[b];
    const int shift = kBlk - min(kBlk, e.y - e.z * kBlk);
    if (row < shift) return;
    const float4* p = reinterpret_cast<const float4*>(is_dk ? a.dk_parts : a.dv_parts) +
                      part_at<D>((int64_t)unit * a.parts, c8 * 2, row);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    for (int k = 0; k < a.parts; ++k, p += kBlk * (D / 4)) {
        const float4 x = p[0], y = p[kBlk];
        v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w, v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
    }
    const float f = is_dk ? a.scale : 1.0f;
    const R97bHeadRows& o = is_dk ? a.dk : a.dv;
    const int64_t tok = (int64_t)e.x + e.z * kBlk + row - shift;
    *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(o.ptr) + tok * o.tok + h * o.head + c8 * 8) =
        make_uint4(pack_bf16(v[0] * f, v[1] * f), pack_bf16(v[2] * f, v[3] * f), pack_bf16(v[4] * f, v[5] * f),
                   pack_bf16(v[6] * f, v[7] * f));
}

// How the key blocks' units are split over their query heads: a block takes as many tiles as its query blocks times the
// group's heads, and the longest unit bounds the pass where the SMs' average share is less. The blocks (a prefix of the
// longest-first table) whose units are above 1.15 of that share go to `parts` units each, with their f32 sums in the
// workspace and one more launch to add them. Measured, dK and dV with the sums: a chat batch of 8192 tokens, 16/4 heads of
// 256: 177 us at 1.15, 181 at 1.25, 179 at 1, 196 at 0.8, 213 at 0.6; of 16384 tokens, 8/2 heads of 128: 66.3, 67.8, 66.6, 74, 79;
// 2 x 4096 tokens, whose longest unit is 1.12 of the share: 517 us unsplit, 528 split (power, not the longest unit, bounds it).
// The whole backward unsplit and by this rule, captured (runs differ by 5 %): 16/4 heads of 256, one token 31.6, 24.1 us,
// turns of 1, 9 and 130 46.9, 32.3, 20 turns of 16 to 400 (ratio 1.35) 105, 113, 4096 + 2 x 2048 (1.48) 739, 662; 16/2 heads,
// 6000 tokens (3.1) 1647, 1016; of 128, 8/2 heads, the 20 turns (2.7) 42.7, 43.4; 8/1 heads, 3 x 4096 (3.0) 558, 350. At
// ratios of 1.02 to 1.14 (8 x 1024, 4 x 2048, 2 x 4096, 8192; both head dims) unsplit and split from 1 on are within 5 %
// of one another, either way.
struct Split {
    int blocks, parts, first;
};
Split split_of(const R97bPacked& p, int Hq, int Hkv) {
    const int grp = Hq / Hkv;
    if (grp == 1 || p.T == 0) return Split{0, 1, 0};
    auto queries = [&](int b) {
        const int32_t* e = p.k_blocks_host + 4 * (int64_t)b;
        return ((int64_t)e[1] + kBlk - 1) / kBlk - e[2];
    };
    int64_t tiles = 0;
    for (int b = 0; b < p.n_blocks; ++b) tiles += queries(b);
    const double limit = 1.15 * (double)(tiles * Hq) / num_sms();
    const double longest = (double)(queries(0) * grp);
    if (longest <= limit) return Split{0, 1, 0};
    Split s{0, grp, 0};
    for (int d = grp - 1; d > 1; --d)
        if (grp % d == 0 && longest / d <= limit) s.parts = d;
    while (s.blocks < p.n_blocks && (double)(queries(s.blocks) * grp) > limit) ++s.blocks;
    while (s.blocks + s.first < p.n_blocks && queries(s.blocks + s.first) * s.parts > queries(0)) ++s.first;
    return s;
}
int64_t part_floats(const Split& s, int Hkv, int D) { return (int64_t)s.blocks * s.parts * Hkv * kBlk * D; }

template <int D, int KIND>
int launch_bwd(const R97bPacked& p, const R97bAttnPackedBwd& a, float* delta, const Split& split, int tail, float* dv_parts,
               float* dk_parts, cudaStream_t st) {
    using C = BCfg<D, KIND>;
    static_assert(C::kSmemBytes <= 232448, "shared memory");
    const bool dq = KIND == kDQ;
    // the rows' operands, the columns' and the accumulating products'
    const R97bHeadRows &a0 = dq ? a.q : a.k, &a1 = dq ? a.dout : a.v, &b0 = dq ? a.k : a.q, &b1 = dq ? a.v : a.dout;
    const R97bHeadRows& c0 = dq ? a.k : (KIND == kDK ? a.q : a.dout);  // (kWhole: the accumulating products reuse b0, b1)
    const int ha = dq ? a.Hq : a.Hkv, hb = dq ? a.Hkv : a.Hq;
    CUtensorMap m[5][2];
    auto same = [&](int i, int j) { m[i][0] = m[j][0], m[i][1] = m[j][1]; };
    if (!make_maps(m[0], a0, ha, D, p.T, tail, kBlk) || !make_maps(m[2], b0, hb, D, p.T, tail, kBlk)) return R97B_EINVAL;
    same(1, 0), same(3, 2), same(4, 2);  // where the kind has no such stream
    if (C::kDP && (!make_maps(m[1], a1, ha, D, p.T, tail, kBlk) || !make_maps(m[3], b1, hb, D, p.T, tail, kBlk)))
        return R97B_EINVAL;
    if (!C::kWhole && !make_maps(m[4], c0, hb, D, p.T, tail, C::kVRows)) return R97B_EINVAL;
    const TailMaps tails{m[0][1], m[1][1], m[2][1], m[3][1], m[4][1]};
    BwdArgs r{};
    r.tail_n = tail;
    r.blocks = reinterpret_cast<const int4*>(dq ? p.q_blocks : p.k_blocks);
    r.lse = a.lse, r.ld_lse = a.ld_lse, r.delta = delta, r.ld_delta = delta_ld(p.T);
    const R97bHeadRows &o0 = dq ? a.dq : (KIND == kDK ? a.dk : a.dv), &o1 = a.dk;
    r.o = reinterpret_cast<const __nv_bfloat16*>(a.o.ptr), r.o_tok = a.o.tok, r.o_head = a.o.head;
    r.out0 = reinterpret_cast<__nv_bfloat16*>(o0.ptr), r.tok0 = o0.tok, r.head0 = o0.head;
    r.out1 = reinterpret_cast<__nv_bfloat16*>(o1.ptr), r.tok1 = o1.tok, r.head1 = o1.head;
    r.a0_head = (int32_t)a0.head, r.a1_head = (int32_t)a1.head, r.b0_head = (int32_t)b0.head, r.b1_head = (int32_t)b1.head;
    r.c0_head = (int32_t)c0.head;
    r.T = (int32_t)p.T;
    auto rows = [](const R97bHeadRows& x) { return reinterpret_cast<const __nv_bfloat16*>(x.ptr); };
    r.a0 = rows(a0), r.a1 = rows(a1), r.b0 = rows(b0), r.b1 = rows(b1), r.c0 = rows(c0);
    r.a0_tok = a0.tok, r.a1_tok = a1.tok, r.b0_tok = b0.tok, r.b1_tok = b1.tok, r.c0_tok = c0.tok;
    r.heads = ha, r.grp = a.Hq / a.Hkv;
    r.split_blocks = dq ? 0 : split.blocks, r.parts = split.parts, r.first_blocks = dq ? 0 : split.first;
    r.part0 = KIND == kDK ? dk_parts : dv_parts, r.part1 = dk_parts;
    r.sl2 = a.scale * kLog2e, r.scale = a.scale;
    const int units = (p.n_blocks + (dq ? 0 : split.blocks * (split.parts - 1))) * ha;
    if (!smem_opt_in(bwd_kernel<D, KIND>, C::kSmemBytes)) return R97B_ELAUNCH;
    bwd_kernel<D, KIND><<<units, kThreads, C::kSmemBytes, st>>>(m[0][0], m[1][0], m[2][0], m[3][0], m[4][0], tails, r);
    return launch_status();
}

template <int D>
int run_bwd(const R97bPacked& p, const R97bAttnPackedBwd& a, cudaStream_t st) {
    float* delta = reinterpret_cast<float*>(a.ws);
    const Split split = split_of(p, a.Hq, a.Hkv);
    const int tail = tail_tokens(p);
    float* dv_parts = delta + a.Hq * delta_ld(p.T);
    float* dk_parts = dv_parts + part_floats(split, a.Hkv, D);
    int rc = launch_bwd<D, kDQ>(p, a, delta, split, tail, dv_parts, dk_parts, st);
    if (rc == R97B_OK) rc = launch_bwd<D, D == 256 ? kDV : kDKV>(p, a, delta, split, tail, dv_parts, dk_parts, st);
    if (D == 256 && rc == R97B_OK) rc = launch_bwd<D, D == 256 ? kDK : kDKV>(p, a, delta, split, tail, dv_parts, dk_parts, st);
    if (split.blocks > 0 && rc == R97B_OK) {
        const SumArgs s{reinterpret_cast<const int4*>(p.k_blocks), dv_parts, dk_parts, a.dv, a.dk, a.scale, a.Hkv,
                        split.parts};
        sum_parts_kernel<D><<<split.blocks * a.Hkv * (2 * kBlk * (D / 8) / 256), 256, 0, st>>>(s);
        rc = launch_status();
    }
    return rc;
}

bool plan_ok(const R97bPacked* p) {
    if (!p || p->n_seq < 0 || p->n_blocks < 0 || p->T < 0 || p->T > 0x7FFFFF00) return false;
    if (p->T == 0) return p->n_blocks == 0;
    return p->n_blocks >= (p->T + 127) / 128 && p->n_blocks <= p->T && p->q_blocks && p->k_blocks && p->k_blocks_host &&
           !(reinterpret_cast<uintptr_t>(p->q_blocks) & 15) && !(reinterpret_cast<uintptr_t>(p->k_blocks) & 15);
}
bool heads_ok(int32_t Hq, int32_t Hkv, int32_t D) {
    return Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && Hq <= 65535 && (D == 128 || D == 256);
}
// Whether an output starts where another operand does (a result is written while others still read).
template <int N>
bool aliased(const void* out, const void* const (&others)[N]) {
    for (const void* o : others)
        if (o == out) return true;
    return false;
}
bool units_ok(const R97bPacked* p, int32_t H) { return (int64_t)p->n_blocks * H <= 0x3FFFFF; }
bool lse_ok(const float* lse, int64_t ld, int64_t T) { return lse && !(reinterpret_cast<uintptr_t>(lse) & 3) && ld >= T; }

}  // namespace
}  // namespace r97b

extern "C" int32_t r97b_packed_blocks(const int32_t* cu_host, int32_t n_seq, int32_t* q_blocks_host,
                                      int32_t* k_blocks_host) {
    if (!cu_host || n_seq < 0 || cu_host[0] != 0) return -1;
    struct Block {
        int32_t tok0, len, i, cost;
    };
    int64_t n = 0;
    for (int32_t s = 0; s < n_seq; ++s) {
        if (cu_host[s + 1] < cu_host[s]) return -1;
        n += ((int64_t)cu_host[s + 1] - cu_host[s] + 127) / 128;
    }
    if (n > 0x7FFFFFFF) return -1;
    std::vector<Block> b;
    try {
        b.reserve((size_t)n);
    } catch (...) {  // no exception crosses the C boundary
        return -1;
    }
    for (int pass = 0; pass < 2; ++pass) {
        int32_t* out = pass == 0 ? q_blocks_host : k_blocks_host;
        if (!out) continue;
        b.clear();
        for (int32_t s = 0; s < n_seq; ++s) {
            const int32_t len = cu_host[s + 1] - cu_host[s], nb = (int32_t)(((int64_t)len + 127) / 128);
            for (int32_t i = 0; i < nb; ++i) b.push_back({cu_host[s], len, i, pass == 0 ? i + 1 : nb - i});
        }
        std::sort(b.begin(), b.end(), [](const Block& x, const Block& y) {
            return x.cost != y.cost ? x.cost > y.cost : (x.tok0 != y.tok0 ? x.tok0 < y.tok0 : x.i < y.i);
        });
        for (size_t i = 0; i < b.size(); ++i) {
            const int32_t row[4] = {b[i].tok0, b[i].len, b[i].i, 0};
            memcpy(out + 4 * i, row, sizeof(row));
        }
    }
    return (int32_t)n;
}

extern "C" int r97b_attn_packed_fwd(const R97bPacked* p, const R97bAttnPackedFwd* a, void* stream) {
    using namespace r97b;
    if (!plan_ok(p) || !a || !heads_ok(a->Hq, a->Hkv, a->D)) return R97B_EINVAL;
    if (!head_rows_ok(a->q, a->Hq, a->D) || !head_rows_ok(a->k, a->Hkv, a->D) || !head_rows_ok(a->v, a->Hkv, a->D) ||
        !head_rows_ok(a->o, a->Hq, a->D) || !lse_ok(a->lse, a->ld_lse, p->T) || !units_ok(p, a->Hq))
        return R97B_EINVAL;
    if (p->T == 0) return R97B_OK;
    if (aliased(a->o.ptr, {a->q.ptr, a->k.ptr, a->v.ptr, a->lse})) return R97B_EINVAL;
    cudaStream_t st = as_stream(stream);
    return a->D == 256 ? launch_fwd<256>(*p, *a, st) : launch_fwd<128>(*p, *a, st);
}

extern "C" int64_t r97b_attn_packed_bwd_workspace_bytes(const R97bPacked* p, int32_t Hq, int32_t Hkv, int32_t D) {
    if (!r97b::plan_ok(p) || !r97b::heads_ok(Hq, Hkv, D)) return -1;
    const r97b::Split s = r97b::split_of(*p, Hq, Hkv);
    return ((int64_t)Hq * r97b::delta_ld(p->T) + 2 * r97b::part_floats(s, Hkv, D)) * 4;
}

extern "C" int r97b_attn_packed_bwd(const R97bPacked* p, const R97bAttnPackedBwd* a, void* stream) {
    using namespace r97b;
    if (!plan_ok(p) || !a || !heads_ok(a->Hq, a->Hkv, a->D)) return R97B_EINVAL;
    if (!head_rows_ok(a->q, a->Hq, a->D) || !head_rows_ok(a->k, a->Hkv, a->D) || !head_rows_ok(a->v, a->Hkv, a->D) ||
        !head_rows_ok(a->o, a->Hq, a->D) || !head_rows_ok(a->dout, a->Hq, a->D) || !head_rows_ok(a->dq, a->Hq, a->D) ||
        !head_rows_ok(a->dk, a->Hkv, a->D) || !head_rows_ok(a->dv, a->Hkv, a->D) || !lse_ok(a->lse, a->ld_lse, p->T) ||
        !units_ok(p, a->Hq))
        return R97B_EINVAL;
    const int64_t need = r97b_attn_packed_bwd_workspace_bytes(p, a->Hq, a->Hkv, a->D);
    if (need < 0 || a->ws_bytes < need || (need > 0 && !a->ws) || (reinterpret_cast<uintptr_t>(a->ws) & 255)) return R97B_EINVAL;
    if (p->T == 0) return R97B_OK;
    for (const void* out : {(const void*)a->dq.ptr, (const void*)a->dk.ptr, (const void*)a->dv.ptr, (const void*)a->ws})
        if (aliased(out, {a->q.ptr, a->k.ptr, a->v.ptr, a->o.ptr, a->dout.ptr, a->lse})) return R97B_EINVAL;
    if (aliased(a->dq.ptr, {a->dk.ptr, a->dv.ptr, a->ws}) || aliased(a->dk.ptr, {a->dv.ptr, a->ws}) || a->dv.ptr == a->ws)
        return R97B_EINVAL;
    cudaStream_t st = as_stream(stream);
    return a->D == 256 ? run_bwd<256>(*p, *a, st) : run_bwd<128>(*p, *a, st);
}
