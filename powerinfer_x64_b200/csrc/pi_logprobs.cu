// Log probabilities of given tokens, entropy and the most likely alternatives, from one
// pass over each row of logits (no reference counterpart: its quality benchmark compares
// whole logit vectors on the host, src/benchmark/mod.rs:45-240).
//
// With m = max x, s = sum e^(x - m) and w = sum (x - m) e^(x - m) over a row:
//   log p(v) = (x_v - m) - log s,      H = -sum p log p = log s - w / s.
// Both terms of H are non-negative, so nothing cancels. A thread keeps (m, s, w) of its
// share and rescales them when its maximum rises (with D = m - m' <= 0:
// s' = s e^D, w' = (w + D s) e^D); shares are joined by the same rule.
//
// Bound: the bytes of the logits (an exponential, four FP32 operations and a compare per
// value; the exponentials alone would allow 148 SMs x 16 / clock, 2.7 times the rate at
// which f32 logits arrive). A row is split over the C CTAs of a cluster where there are
// few rows, and their results join through distributed shared memory: one launch, no
// workspace, no atomics on memory, so calls and captured graphs share nothing.
#include "pi_common.cuh"
#include "pi_internal.h"

#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <exception>
#include <map>

namespace cg = cooperative_groups;

namespace {

constexpr int LP_NT = 256;       // threads of a CTA
constexpr int LP_W = LP_NT / 32;
constexpr int LP_U = 2;          // 16-byte loads of a step; the next step's are in flight
constexpr int LP_OCC = 4;        // CTAs of an SM
constexpr int LP_MAXC = 16;      // CTAs of a cluster at most
constexpr int LP_MAXTOP = 32;    // alternatives at most
constexpr float LP_LOG2E = 1.4426950408889634f;
constexpr float LP_LOWEST = -3.402823466e38f;

struct LogprobArgs {
    const void* logits;
    int64_t T, V, ld;
    const int64_t* targets;
    int64_t n_targets;
    int n_top, C;
    float* logp;
    float* entropy;
    int32_t* top_ids;
    float* top_logp;
    uint32_t* err;
};

struct LpStat {
    float m, s, w;
};

PI_DEV float ex2(float a) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a));
    return r;
}
// x - m for x <= m, held above -200 (e^-200 is 0 in f32), so that a masked value (-inf or
// the type's lowest) adds 0 to both sums instead of 0 * inf; NaN stays NaN.
PI_DEV float lp_shift(float x, float m) { return max_nan(x - m, -200.0f); }

PI_DEV void lp_join(LpStat& a, const LpStat& b) {
    const float m = fmaxf(a.m, b.m);
    const float da = lp_shift(a.m, m), db = lp_shift(b.m, m);
    const float ea = ex2(da * LP_LOG2E), eb = ex2(db * LP_LOG2E);
    a.w = fmaf(da, a.s, a.w) * ea + fmaf(db, b.s, b.w) * eb;
    a.s = a.s * ea + b.s * eb;
    a.m = m;
}

template <int N>
PI_DEV float lp_max(const float* f) {
    float a = fmaxf(f[0], f[1]), b = fmaxf(f[2], f[3]);
    if constexpr (N == 8) {
        a = fmaxf(a, fmaxf(f[4], f[5]));
        b = fmaxf(b, fmaxf(f[6], f[7]));
    }
    return fmaxf(a, b);
}

// One 64-bit key per value: larger for a larger logit and, where they tie (-0 and 0 too),
// for a lower index. 0 stands for no value; values above -inf have keys above 0.
PI_DEV uint64_t lp_key(float v, uint32_t i) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return ((uint64_t)((b & 0x80000000u) ? ~b : (b | 0x80000000u)) << 32) | (uint32_t)~i;
}
PI_DEV uint32_t lp_key_index(uint64_t k) { return ~(uint32_t)k; }
PI_DEV float lp_key_value(uint64_t k) {
    const uint32_t h = (uint32_t)(k >> 32);
    return __uint_as_float((h & 0x80000000u) ? (h ^ 0x80000000u) : ~h);
}
PI_DEV uint64_t warp_max_key(uint64_t k) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
    return ((uint64_t)hi << 32) | lo;
}

PI_DEV float lp_float(float v) { return v; }
PI_DEV float lp_float(__half v) { return __half2float(v); }
PI_DEV float lp_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename ET>
PI_DEV void lp_unpack(const int4& q, float* x) {
    if constexpr (sizeof(ET) == 4) {
        x[0] = __int_as_float(q.x);
        x[1] = __int_as_float(q.y);
        x[2] = __int_as_float(q.z);
        x[3] = __int_as_float(q.w);
    } else {
        const uint32_t r[4] = {(uint32_t)q.x, (uint32_t)q.y, (uint32_t)q.z, (uint32_t)q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same_v<ET, __half>) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r[i]));
                x[2 * i] = f.x;
                x[2 * i + 1] = f.y;
            } else {  // bf16 is the upper half of an f32
                x[2 * i] = __uint_as_float(r[i] << 16);
                x[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
            }
        }
    }
}

// The largest values a warp has seen so far: a shared buffer of keys, a count, and the
// value a further one has to exceed. Once n values of lower index reach `thr`, a later
// value that only ties cannot be among the n best, so the comparison is strict; `incl`
// admits ties for as long as that is not so.
template <int CAP>
struct LpTop {
    uint64_t* buf;
    int cnt = 0, n, lane;
    float thr = -INFINITY;
    bool incl = false;

    // keeps the n best of the buffer, in order
    PI_DEV void compact() {
        constexpr int P = CAP / 32;
        uint64_t k[P];
#pragma unroll
        for (int i = 0; i < P; ++i) k[i] = lane + 32 * i < cnt ? buf[lane + 32 * i] : 0;
        __syncwarp();
        const int keep = min(n, cnt);
        uint64_t best = 0;
        for (int r = 0; r < keep; ++r) {
            uint64_t mine = 0;
#pragma unroll
            for (int i = 0; i < P; ++i) mine = k[i] > mine ? k[i] : mine;
            best = warp_max_key(mine);
#pragma unroll
            for (int i = 0; i < P; ++i) k[i] = k[i] == best ? 0 : k[i];  // keys are distinct
            if (lane == 0) buf[r] = best;
        }
        cnt = keep;
        if (keep == n) {
            thr = fmaxf(thr, lp_key_value(best));
            incl = false;
        }
        __syncwarp();
    }
    PI_DEV bool passes(float x) const { return x > thr || (incl && x == thr); }
    // N values per lane, index i0 + j; every lane calls it
    template <int N>
    PI_DEV void add(const float* x, float vmax, uint32_t i0) {
        if (!__any_sync(0xffffffffu, passes(vmax))) return;
        if (cnt + 32 * N > CAP) compact();
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const bool in = passes(x[j]);
            const uint32_t b = __ballot_sync(0xffffffffu, in);
            if (in) buf[cnt + __popc(b & ((1u << lane) - 1u))] = lp_key(x[j], i0 + j);
            cnt += __popc(b);
        }
        __syncwarp();
    }
};

// The n best of `cnt` distinct keys in `all` to best[0..n) (0 where there are fewer): a
// key's place is the number of larger ones, counted by four lanes.
PI_DEV void lp_rank(const uint64_t* all, int cnt, uint64_t* best, int n, int tid) {
    if (tid < n && tid >= cnt) best[tid] = 0;
    for (int i0 = 0; i0 < cnt; i0 += LP_NT / 4) {
        const int i = i0 + (tid >> 2);
        const uint64_t k = i < cnt ? all[i] : ~0ull;
        int r = 0;
        for (int j = tid & 3; j < cnt; j += 4) r += all[j] > k;
        r += __shfl_xor_sync(0xffffffffu, r, 1);
        r += __shfl_xor_sync(0xffffffffu, r, 2);
        if (i < cnt && r < n && (tid & 3) == 0) best[r] = k;
    }
}

// Joins the states of the lanes whose numbers differ below `width`, a power of two.
PI_DEV void lp_join_lanes(LpStat& st, int width) {
    for (int o = width >> 1; o > 0; o >>= 1) {
        LpStat b;
        b.m = __shfl_xor_sync(0xffffffffu, st.m, o);
        b.s = __shfl_xor_sync(0xffffffffu, st.s, o);
        b.w = __shfl_xor_sync(0xffffffffu, st.w, o);
        lp_join(st, b);
    }
}

// Row blockIdx.x / C, share blockIdx.x % C. The first LP_U loads of a thread give, over
// groups of four lanes, 64 maxima: the n-th largest of them is reached by n values at
// least, so only what reaches it is kept from the start (about n values of the first
// 2048 or 4096, then n / i of the i-th step), and the buffers hardly ever fill.
template <typename ET, bool TOP>
__global__ __launch_bounds__(LP_NT, LP_OCC) void k_token_logprobs(const LogprobArgs a) {
    constexpr int NV = 16 / (int)sizeof(ET);
    constexpr int CAP = 64 + 32 * NV;  // n kept after compact() and one load of every lane
    __shared__ uint64_t s_buf[TOP ? LP_W * CAP : 1];
    __shared__ uint64_t s_all[TOP ? LP_MAXC * LP_MAXTOP : 1];
    __shared__ uint64_t s_lists[TOP ? LP_MAXC * LP_MAXTOP : 1];  // the cluster's lists, in its first CTA
    __shared__ LpStat s_stats[LP_MAXC];                          // and its states
    __shared__ uint64_t s_best[LP_MAXTOP];
    __shared__ LpStat s_stat[LP_W], s_cta;
    __shared__ float s_max[64], s_thr;
    __shared__ int s_cnt[LP_W];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int C = a.C;
    const int64_t row = blockIdx.x / C;
    const int rank = (int)(blockIdx.x - row * C);
    const ET* x = reinterpret_cast<const ET*>(a.logits) + row * a.ld;
    // values before the first 16-byte boundary and after the last whole 16 bytes are read
    // one by one by the first warp of the row
    const int64_t head = min((int64_t)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(ET)), a.V);
    const int64_t nvec = (a.V - head) / NV, tail = head + nvec * NV;
    const int4* xv = reinterpret_cast<const int4*>(x + head);
    const int64_t step = (int64_t)C * LP_NT;
    const bool edges = rank == 0 && warp == 0;
    // the first CTA of the cluster must run before the others write into its shared memory
    if (C > 1) cluster_arrive();

    LpStat st{LP_LOWEST, 0.0f, 0.0f};
    auto scalar = [&](float v) {
        if (v > st.m) {
            const float dm = lp_shift(st.m, v), e = ex2(dm * LP_LOG2E);
            st.w = fmaf(dm, st.s, st.w) * e;
            st.s *= e;
            st.m = v;
        }
        const float t = lp_shift(v, st.m), e = ex2(t * LP_LOG2E);
        st.s += e;
        st.w = fmaf(t, e, st.w);
    };
    LpTop<CAP> top;
    if constexpr (TOP) {
        top.buf = s_buf + warp * CAP;
        top.n = a.n_top;
        top.lane = lane;
    }
    if (edges) {
        const float v = lane < head ? lp_float(x[lane]) : -INFINITY;
        if (lane < head) scalar(v);
        if constexpr (TOP) top.template add<1>(&v, v, (uint32_t)lane);
    }
    // the next LP_U loads are on their way while the current ones are worked on
    int4 q[LP_U], qn[LP_U];
    int64_t v0 = (int64_t)rank * LP_NT + tid;
#pragma unroll
    for (int u = 0; u < LP_U; ++u)
        if (v0 + u * step < nvec) qn[u] = ld_stream(xv + v0 + u * step);
    bool first = true;
    for (; v0 - tid < nvec || first; v0 += LP_U * step) {
#pragma unroll
        for (int u = 0; u < LP_U; ++u) {
            q[u] = qn[u];
            if (v0 + (LP_U + u) * step < nvec) qn[u] = ld_stream(xv + v0 + (LP_U + u) * step);
        }
        if constexpr (TOP) {
            if (first) {
                float mx = -INFINITY;
#pragma unroll
                for (int u = 0; u < LP_U; ++u)
                    if (v0 + u * step < nvec) {
                        float f[NV];
                        lp_unpack<ET>(q[u], f);
                        mx = fmaxf(mx, lp_max<NV>(f));
                    }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                if ((lane & 3) == 0) s_max[tid >> 2] = mx;
                __syncthreads();
                {
                    const int i = tid >> 2;  // four lanes count the maxima above the i-th
                    const float mine = s_max[i];
                    int r = 0;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int o = (tid & 3) + 4 * j;
                        r += s_max[o] > mine || (s_max[o] == mine && o < i);
                    }
                    r += __shfl_xor_sync(0xffffffffu, r, 1);
                    r += __shfl_xor_sync(0xffffffffu, r, 2);
                    if (r == a.n_top - 1) s_thr = mine;
                }
                __syncthreads();
                top.thr = s_thr;
                top.incl = s_thr > -INFINITY;
            }
        }
#pragma unroll
        for (int u = 0; u < LP_U; ++u) {
            const bool live = v0 + u * step < nvec;
            float f[NV];
            float vmax = -INFINITY;
            if (live) {
                lp_unpack<ET>(q[u], f);
                vmax = lp_max<NV>(f);
                if (vmax > st.m) {
                    const float dm = lp_shift(st.m, vmax), e = ex2(dm * LP_LOG2E);
                    st.w = fmaf(dm, st.s, st.w) * e;
                    st.s *= e;
                    st.m = vmax;
                }
                const uint64_t m2 = pack2(-st.m, -st.m), l2 = pack2(LP_LOG2E, LP_LOG2E);
                uint64_t s2 = 0, w2 = 0;
#pragma unroll
                for (int j = 0; j < NV; j += 2) {
                    float2 t = unpack2(add2(pack2(f[j], f[j + 1]), m2));
                    t.x = max_nan(t.x, -200.0f);
                    t.y = max_nan(t.y, -200.0f);
                    const uint64_t tt = pack2(t.x, t.y);
                    const float2 g = unpack2(mul2(tt, l2));
                    const uint64_t e = pack2(ex2(g.x), ex2(g.y));
                    s2 = add2(s2, e);
                    w2 = fma2(tt, e, w2);
                }
                const float2 sp = unpack2(s2), wp = unpack2(w2);
                st.s += sp.x + sp.y;
                st.w += wp.x + wp.y;
            } else {
#pragma unroll
                for (int j = 0; j < NV; ++j) f[j] = -INFINITY;
            }
            if constexpr (TOP) top.template add<NV>(f, vmax, (uint32_t)(head + (v0 + u * step) * NV));
        }
        if constexpr (TOP) top.incl = false;
        first = false;
    }
    if (edges) {
        const int64_t i = tail + lane;
        const float v = i < a.V ? lp_float(x[i]) : -INFINITY;
        if (i < a.V) scalar(v);
        if constexpr (TOP) top.template add<1>(&v, v, (uint32_t)i);
    }

    // join: lanes, warps, then the CTAs of the cluster
    lp_join_lanes(st, 32);
    if (lane == 0) s_stat[warp] = st;
    if constexpr (TOP) {
        if (lane == 0) s_cnt[warp] = top.cnt;
        __syncthreads();
        int total = 0;
        for (int i = 0; i < LP_W; ++i) total += s_cnt[i];
        if (total > LP_NT) {
            __syncthreads();
            if (top.cnt > a.n_top) top.compact();
            if (lane == 0) s_cnt[warp] = top.cnt;
            __syncthreads();
        }
        int at = 0;
        total = 0;
        for (int i = 0; i < LP_W; ++i) {
            if (i < warp) at += s_cnt[i];
            total += s_cnt[i];
        }
        for (int i = lane; i < top.cnt; i += 32) s_all[at + i] = top.buf[i];
        __syncthreads();
        lp_rank(s_all, total, s_best, a.n_top, tid);
    } else {
        __syncthreads();
    }
    if (warp == 0) {
        LpStat t = s_stat[lane % LP_W];
        lp_join_lanes(t, LP_W);
        if (lane == 0) s_cta = t;
    }
    if (C > 1) {
        __syncthreads();
        cluster_wait();
        cg::cluster_group cl = cg::this_cluster();
        if (tid == 0) *cl.map_shared_rank(&s_stats[rank], 0) = s_cta;
        if constexpr (TOP)
            if (tid < a.n_top) cl.map_shared_rank(s_lists, 0)[rank * a.n_top + tid] = s_best[tid];
        cluster_arrive();
        if (rank != 0) return;
        cluster_wait();
        if (warp == 0) {
            LpStat t = s_stats[lane % C];
            lp_join_lanes(t, C);
            if (lane == 0) s_cta = t;
        }
        if constexpr (TOP) {
            // ceil(n / C) values of every CTA reach the least of the CTAs' ceil(n / C)-th ones, n
            // values at least: only what reaches it is ranked
            const int deep = (a.n_top + C - 1) / C;
            if (tid == 0) s_cnt[0] = 0;
            __syncthreads();
            uint64_t bound = lane < C ? s_lists[lane * a.n_top + deep - 1] : ~0ull;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const uint64_t other = __shfl_xor_sync(0xffffffffu, bound, o);
                bound = other < bound ? other : bound;
            }
            for (int i = tid; i < C * a.n_top; i += LP_NT)
                if (s_lists[i] >= bound && s_lists[i]) s_all[atomicAdd(&s_cnt[0], 1)] = s_lists[i];
            __syncthreads();
            lp_rank(s_all, s_cnt[0], s_best, a.n_top, tid);
        }
    }
    __syncthreads();
    const LpStat t = s_cta;
    // s == 0: the row's mask leaves nothing; s NaN: a NaN or +inf, no distribution
    const bool none = t.s == 0.0f, bad = t.s != t.s;
    const float log_s = none ? 0.0f : logf(t.s), nan = __int_as_float(0x7fffffff);
    if (tid == 0 && a.entropy) a.entropy[row] = none ? 0.0f : (bad ? nan : log_s - t.w / t.s);
    for (int64_t j = tid; j < a.n_targets; j += LP_NT) {
        const int64_t v = a.targets[row * a.n_targets + j];
        float r = 0.0f;  // a negative target is no token
        if (v >= a.V) {
            atomicOr(a.err, PI_DEVERR_INDEX);
            r = nan;
        } else if (v >= 0) {
            const float xt = lp_float(x[v]);
            r = none ? -INFINITY : (bad ? nan : (xt - t.m) - log_s);
        }
        a.logp[row * a.n_targets + j] = r;
    }
    if constexpr (TOP) {
        if (tid < a.n_top) {
            const uint64_t k = bad ? 0 : s_best[tid];
            a.top_ids[row * a.n_top + tid] = k ? (int32_t)lp_key_index(k) : -1;
            a.top_logp[row * a.n_top + tid] = bad ? nan : (k ? (lp_key_value(k) - t.m) - log_s : -INFINITY);
        }
    }
}

// Clusters of more than 8 CTAs need the kernel's consent, once per kernel and device.
cudaError_t allow_wide_cluster(const void* fn, int device) {
    static std::mutex mu;
    static std::map<std::pair<const void*, int>, bool> done;
    std::lock_guard<std::mutex> g(mu);
    bool& have = done[{fn, device}];
    if (have) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    have = e == cudaSuccess;
    return e;
}

template <typename ET>
cudaError_t launch_logprobs(pi_ctx* ctx, const LogprobArgs& a, cudaStream_t st) {
    auto kern = a.n_top > 0 ? k_token_logprobs<ET, true> : k_token_logprobs<ET, false>;
    if (a.C > 8)
        if (cudaError_t e = allow_wide_cluster((const void*)kern, ctx->device)) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.T * a.C));
    cfg.blockDim = dim3(LP_NT);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)a.C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = a.C > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

int token_logprobs(pi_ctx* ctx, const void* logits, int32_t dtype, int64_t T, int64_t V, int64_t ld,
                   const int64_t* targets, int64_t n_targets, int32_t n_top, float* logp, float* entropy,
                   int32_t* top_ids, float* top_logp, cudaStream_t st) {
    const int es = dtype == PI_QT_F32 ? 4 : 2;
    if (dtype != PI_QT_F32 && dtype != PI_QT_F16 && dtype != PI_QT_BF16)
        return pi_set_error(ctx, PI_ERR_ARG, "logprobs: logits must be F32, F16 or BF16");
    if (T < 0 || V < 1 || V > INT32_MAX || T > (1 << 24) || n_targets < 0 || n_targets > (1 << 20))
        return pi_set_error(ctx, PI_ERR_ARG, "logprobs: need 0 <= T <= 2^24 rows of 1 <= V < 2^31 logits, at most 2^20 targets a row");
    if (n_top < 0 || n_top > LP_MAXTOP)
        return pi_set_error(ctx, PI_ERR_ARG, "logprobs: 0 <= n_top <= 32");
    if (T == 0) return PI_OK;
    if (!logits || ld < 0 || (n_targets && (!targets || !logp)) || (n_top && (!top_ids || !top_logp)))
        return pi_set_error(ctx, PI_ERR_ARG, "logprobs: null pointer or negative row stride");
    if ((uintptr_t)logits % es) return pi_set_error(ctx, PI_ERR_ARG, "logprobs: logits are not aligned to their type");
    PiDeviceGuard dev(ctx->device);
    LogprobArgs a{logits, T, V, ld, targets, n_targets, n_top, 1, logp, entropy, top_ids, top_logp, ctx->dev_err};
    // CTAs of a row: as long as all of the grid's run at once and each has two loads a thread
    const int64_t nvec = V * es / 16, sms = ctx->sm_count > 0 ? ctx->sm_count : 148;
    while (a.C < LP_MAXC && T * a.C * 2 <= LP_OCC * sms && nvec >= (int64_t)a.C * 2 * 2 * LP_NT) a.C *= 2;
    PiProfScope ps(ctx, st, "k_token_logprobs");
    const cudaError_t e = dtype == PI_QT_F32   ? launch_logprobs<float>(ctx, a, st)
                          : dtype == PI_QT_F16 ? launch_logprobs<__half>(ctx, a, st)
                                               : launch_logprobs<__nv_bfloat16>(ctx, a, st);
    return pi_cuda_check(ctx, e, "logprobs");
}

}  // namespace

extern "C" int pi_token_logprobs(pi_ctx* ctx, const void* logits, int32_t dtype, int64_t T, int64_t V, int64_t ld,
                                 const int64_t* targets, int64_t n_targets, int32_t n_top, float* logp,
                                 float* entropy, int32_t* top_ids, float* top_logp, void* stream) {
    if (!ctx) return PI_ERR_ARG;
    try {
        return token_logprobs(ctx, logits, dtype, T, V, ld, targets, n_targets, n_top, logp, entropy, top_ids,
                              top_logp, (cudaStream_t)stream);
    } catch (const std::exception&) {  // an allocation of the host failed
        return PI_ERR_OOM;
    }
}
