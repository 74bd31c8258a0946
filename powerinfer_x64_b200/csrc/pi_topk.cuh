// Routing of one token by one warp from its exact logits (model/mod.rs:1278-1312).
#pragma once
#include "pi_common.cuh"

// Top-k by probability with ties to the lowest expert index: a round takes the
// largest key with redux.sync max (keys: probability bits + 2, order-preserving
// for non-negative floats; 1 for NaN, 0 for taken) and then the lowest index
// holding it with redux.sync min.
// The logits are read past L1: other CTAs may have written them.
template <int NPL>
PI_DEV void topk_token(const float* __restrict__ logits, int t, int E, int k, int has_shgate,
                       int32_t* __restrict__ idx, float* __restrict__ gates, float* __restrict__ shscale,
                       int32_t* __restrict__ counts, float* p, int* sel, int lane) {
    const float* lr = logits + (size_t)t * (E + 1);
    float l[NPL];
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const int e = lane + 32 * j;
        l[j] = (e < E) ? __ldcg(lr + e) : -INFINITY;
        if (e < E) m = fmaxf(m, l[j]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const int e = lane + 32 * j;
        if (e < E) p[e] = exp_cr(fsub(l[j], m));
    }
    __syncwarp();
    // exp_sum: sequential sum in expert order (model/mod.rs:1282)
    float es = 0.0f;
    if (lane == 0) {
#pragma unroll 16
        for (int e = 0; e < E; ++e) es = fadd(es, p[e]);
    }
    es = __shfl_sync(0xffffffffu, es, 0);
    float pr[NPL];
    uint32_t key[NPL];
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const int e = lane + 32 * j;
        pr[j] = (e < E) ? fdiv(p[e], es) : 0.0f;
        key[j] = (e < E) ? (pr[j] == pr[j] ? __float_as_uint(pr[j]) + 2u : 1u) : 0u;
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const int e = lane + 32 * j;
        if (e < E) p[e] = pr[j];
    }
    for (int r = 0; r < k; ++r) {
        uint32_t mk = 0;
#pragma unroll
        for (int j = 0; j < NPL; ++j) mk = max(mk, key[j]);
        mk = __reduce_max_sync(0xffffffffu, mk);
        uint32_t me = 0xffffffffu;
#pragma unroll
        for (int j = NPL - 1; j >= 0; --j)
            if (key[j] == mk) me = lane + 32 * j;
        const int bi = (int)__reduce_min_sync(0xffffffffu, me);
        if ((bi & 31) == lane) {
#pragma unroll
            for (int j = 0; j < NPL; ++j)
                if (j == (bi >> 5)) key[j] = 0;
        }
        if (lane == 0) sel[r] = bi;
    }
    __syncwarp();
    // ascending sort of the k selected indices (model/mod.rs:1303)
    const int mine = (lane < k) ? sel[lane] : 0x7fffffff;
    int rank = 0;
    for (int r = 0; r < k; ++r) rank += (sel[r] < mine);
    __syncwarp();
    if (lane < k) sel[rank] = mine;
    __syncwarp();
    float ssum = 0.0f;
    if (lane == 0)
        for (int r = 0; r < k; ++r) ssum = fadd(ssum, p[sel[r]]);
    ssum = __shfl_sync(0xffffffffu, ssum, 0);
    if (lane < k) {
        const int e = sel[lane];
        const float pe = p[e];
        idx[(size_t)t * k + lane] = e;
        gates[(size_t)t * k + lane] = (ssum > 0.0f) ? fdiv(pe, ssum) : pe;
        if (counts) atomicAdd(&counts[e], 1);
    }
    if (lane == 0 && shscale) shscale[t] = has_shgate ? sigmoid_ref(__ldcg(lr + E)) : 1.0f;
    __syncwarp();
}
