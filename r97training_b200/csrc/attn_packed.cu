// attn_packed.cu -- causal grouped-query attention over packed (ragged) sequences, forward and the backward that
// recomputes the probabilities (reference: attention_twin and attention_host_adjoint,
// src/adjoint/host/attention.cpp:261-414).
//
//   o_t = sum_{j <= t} p_tj v_j,  p_tj = exp(scale q_t . k_j - lse_t)      over the tokens of t's own sequence
//   dv_j = sum_t p_tj do_t,  ds_tj = p_tj (do_t . v_j - do_t . o_t),  dq_t = scale sum_j ds_tj k_j,
//   dk_j = scale sum_t ds_tj q_t                                          (dk, dv summed over the group's heads)
//
// One warp a row, f32 throughout.
#include "r97b_internal.h"

#include <algorithm>
#include <cuda_bf16.h>
#include <math.h>
#include <string.h>
#include <vector>

namespace r97b {
namespace {

struct Rows {
    __nv_bfloat16* p;
    int64_t tok, head;
    __device__ __nv_bfloat16* at(int64_t t, int h) const { return p + t * tok + (int64_t)h * head; }
};
Rows rows_of(const R97bHeadRows& r) { return Rows{reinterpret_cast<__nv_bfloat16*>(r.ptr), r.tok, r.head}; }

struct Args {
    const int4* blocks;
    Rows q, k, v, o, dout, dq, dk, dv;
    float* lse;
    int64_t ld_lse;
    int32_t Hq, grp;
    float scale;
};

__device__ __forceinline__ float sum32(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}
template <int N>
__device__ __forceinline__ void ld(const __nv_bfloat16* p, float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __bfloat162float(p[32 * i]);
}
template <int N>
__device__ __forceinline__ float dot(const float (&a)[N], const float (&b)[N]) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(a[i], b[i], s);
    return sum32(s);
}

// grid (block, head, 16): 8 warps, one row each
template <int N>
__global__ void __launch_bounds__(256) fwd_simple(const Args a) {
    const int4 b = a.blocks[blockIdx.x];
    const int h = blockIdx.y, lane = threadIdx.x & 31, r = b.z * 128 + blockIdx.z * 8 + (threadIdx.x >> 5);
    if (r >= b.y) return;
    float q[N], o[N], x[N];
    ld<N>(a.q.at(b.x + r, h) + lane, q);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    for (int j = 0; j <= r; ++j) {
        ld<N>(a.k.at(b.x + j, h / a.grp) + lane, x);
        const float s = dot<N>(q, x) * a.scale, mn = fmaxf(m, s);
        const float c = mn == -INFINITY ? 1.0f : expf(m - mn), p = mn == -INFINITY ? 0.0f : expf(s - mn);
        ld<N>(a.v.at(b.x + j, h / a.grp) + lane, x);
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = o[i] * c + p * x[i];
        l = l * c + p;
        m = mn;
    }
    __nv_bfloat16* op = a.o.at(b.x + r, h) + lane;
#pragma unroll
    for (int i = 0; i < N; ++i) op[32 * i] = __float2bfloat16_rn(o[i] / l);
    if (lane == 0) a.lse[h * a.ld_lse + b.x + r] = m + logf(l);
}

template <int N>
__global__ void __launch_bounds__(256) dq_simple(const Args a) {
    const int4 b = a.blocks[blockIdx.x];
    const int h = blockIdx.y, lane = threadIdx.x & 31, r = b.z * 128 + blockIdx.z * 8 + (threadIdx.x >> 5);
    if (r >= b.y) return;
    float q[N], d[N], g[N], x[N], y[N];
    ld<N>(a.q.at(b.x + r, h) + lane, q);
    ld<N>(a.dout.at(b.x + r, h) + lane, d);
    ld<N>(a.o.at(b.x + r, h) + lane, x);
    const float delta = dot<N>(d, x), lse = a.lse[h * a.ld_lse + b.x + r];
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = 0.0f;
    for (int j = 0; j <= r; ++j) {
        ld<N>(a.k.at(b.x + j, h / a.grp) + lane, x);
        ld<N>(a.v.at(b.x + j, h / a.grp) + lane, y);
        const float ds = expf(dot<N>(q, x) * a.scale - lse) * (dot<N>(d, y) - delta);
#pragma unroll
        for (int i = 0; i < N; ++i) g[i] = fmaf(ds, x[i], g[i]);
    }
    __nv_bfloat16* op = a.dq.at(b.x + r, h) + lane;
#pragma unroll
    for (int i = 0; i < N; ++i) op[32 * i] = __float2bfloat16_rn(g[i] * a.scale);
}

// one warp a key row of one key/value head
template <int N>
__global__ void __launch_bounds__(256) dkv_simple(const Args a) {
    const int4 b = a.blocks[blockIdx.x];
    const int g = blockIdx.y, lane = threadIdx.x & 31, j = b.z * 128 + blockIdx.z * 8 + (threadIdx.x >> 5);
    if (j >= b.y) return;
    float k[N], v[N], dk[N], dv[N], x[N], y[N];
    ld<N>(a.k.at(b.x + j, g) + lane, k);
    ld<N>(a.v.at(b.x + j, g) + lane, v);
#pragma unroll
    for (int i = 0; i < N; ++i) dk[i] = dv[i] = 0.0f;
    for (int h = g * a.grp; h < (g + 1) * a.grp; ++h) {
        for (int t = j; t < b.y; ++t) {
            ld<N>(a.q.at(b.x + t, h) + lane, x);
            const float p = expf(dot<N>(x, k) * a.scale - a.lse[h * a.ld_lse + b.x + t]);
            ld<N>(a.dout.at(b.x + t, h) + lane, y);
            float o[N];
            ld<N>(a.o.at(b.x + t, h) + lane, o);
            const float ds = p * (dot<N>(y, v) - dot<N>(y, o));
#pragma unroll
            for (int i = 0; i < N; ++i) {
                dv[i] = fmaf(p, y[i], dv[i]);
                dk[i] = fmaf(ds, x[i], dk[i]);
            }
        }
    }
    __nv_bfloat16* kp = a.dk.at(b.x + j, g) + lane;
    __nv_bfloat16* vp = a.dv.at(b.x + j, g) + lane;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        kp[32 * i] = __float2bfloat16_rn(dk[i] * a.scale);
        vp[32 * i] = __float2bfloat16_rn(dv[i]);
    }
}

bool plan_ok(const R97bPacked* p) {
    if (!p || p->n_seq < 0 || p->n_blocks < 0 || p->T < 0 || p->T > 0x7FFFFF00) return false;
    if (p->T == 0) return p->n_blocks == 0;
    return p->n_blocks >= (p->T + 127) / 128 && p->n_blocks <= p->T && p->q_blocks && p->k_blocks &&
           !(reinterpret_cast<uintptr_t>(p->q_blocks) & 15) && !(reinterpret_cast<uintptr_t>(p->k_blocks) & 15);
}
bool heads_ok(int32_t Hq, int32_t Hkv, int32_t D) {
    return Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && Hq <= 65535 && (D == 128 || D == 256);
}
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
    for (int pass = 0; pass < 2; ++pass) {
        int32_t* out = pass == 0 ? q_blocks_host : k_blocks_host;
        if (!out) continue;
        b.clear();
        b.reserve((size_t)n);
        for (int32_t s = 0; s < n_seq; ++s) {
            const int32_t len = cu_host[s + 1] - cu_host[s], nb = (int32_t)(((int64_t)len + 127) / 128);
            for (int32_t i = 0; i < nb; ++i) b.push_back({cu_host[s], len, i, pass == 0 ? i + 1 : nb - i});
        }
        std::stable_sort(b.begin(), b.end(), [](const Block& x, const Block& y) { return x.cost > y.cost; });
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
        !head_rows_ok(a->o, a->Hq, a->D) || !lse_ok(a->lse, a->ld_lse, p->T))
        return R97B_EINVAL;
    if (p->T == 0) return R97B_OK;
    Args r{};
    r.blocks = reinterpret_cast<const int4*>(p->q_blocks);
    r.q = rows_of(a->q), r.k = rows_of(a->k), r.v = rows_of(a->v), r.o = rows_of(a->o);
    r.lse = a->lse, r.ld_lse = a->ld_lse, r.Hq = a->Hq, r.grp = a->Hq / a->Hkv, r.scale = a->scale;
    const dim3 grid(p->n_blocks, a->Hq, 16);
    if (a->D == 256)
        fwd_simple<8><<<grid, 256, 0, as_stream(stream)>>>(r);
    else
        fwd_simple<4><<<grid, 256, 0, as_stream(stream)>>>(r);
    return launch_status();
}

extern "C" int64_t r97b_attn_packed_bwd_workspace_bytes(const R97bPacked* p, int32_t Hq, int32_t Hkv, int32_t D) {
    if (!r97b::plan_ok(p) || !r97b::heads_ok(Hq, Hkv, D)) return -1;
    return 0;
}

extern "C" int r97b_attn_packed_bwd(const R97bPacked* p, const R97bAttnPackedBwd* a, void* stream) {
    using namespace r97b;
    if (!plan_ok(p) || !a || !heads_ok(a->Hq, a->Hkv, a->D)) return R97B_EINVAL;
    if (!head_rows_ok(a->q, a->Hq, a->D) || !head_rows_ok(a->k, a->Hkv, a->D) || !head_rows_ok(a->v, a->Hkv, a->D) ||
        !head_rows_ok(a->o, a->Hq, a->D) || !head_rows_ok(a->dout, a->Hq, a->D) || !head_rows_ok(a->dq, a->Hq, a->D) ||
        !head_rows_ok(a->dk, a->Hkv, a->D) || !head_rows_ok(a->dv, a->Hkv, a->D) || !lse_ok(a->lse, a->ld_lse, p->T))
        return R97B_EINVAL;
    const int64_t need = r97b_attn_packed_bwd_workspace_bytes(p, a->Hq, a->Hkv, a->D);
    if (need < 0 || a->ws_bytes < need || (need > 0 && !a->ws) || (reinterpret_cast<uintptr_t>(a->ws) & 255)) return R97B_EINVAL;
    if (p->T == 0) return R97B_OK;
    Args r{};
    r.q = rows_of(a->q), r.k = rows_of(a->k), r.v = rows_of(a->v), r.o = rows_of(a->o), r.dout = rows_of(a->dout);
    r.dq = rows_of(a->dq), r.dk = rows_of(a->dk), r.dv = rows_of(a->dv);
    r.lse = const_cast<float*>(a->lse), r.ld_lse = a->ld_lse, r.Hq = a->Hq, r.grp = a->Hq / a->Hkv, r.scale = a->scale;
    cudaStream_t st = as_stream(stream);
    r.blocks = reinterpret_cast<const int4*>(p->q_blocks);
    const dim3 gq(p->n_blocks, a->Hq, 16), gk(p->n_blocks, a->Hkv, 16);
    if (a->D == 256)
        dq_simple<8><<<gq, 256, 0, st>>>(r);
    else
        dq_simple<4><<<gq, 256, 0, st>>>(r);
    r.blocks = reinterpret_cast<const int4*>(p->k_blocks);
    if (a->D == 256)
        dkv_simple<8><<<gk, 256, 0, st>>>(r);
    else
        dkv_simple<4><<<gk, 256, 0, st>>>(r);
    return launch_status(2);
}
