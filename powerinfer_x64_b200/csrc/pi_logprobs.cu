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

constexpr int LP_U = 4;          // 16-byte loads of a step
// NT threads work on a row together: 256 (or a cluster of such CTAs), 64 from five rows per SM on,
// one warp from eight. What does not shrink with the row (threshold, joins, ranking) is then
// paid by fewer warps, and the CTAs fill the SMs in whole waves: 2048 rows of 32000 bf16 take 36 us
// with a warp, 41 with 256 threads; 1000 rows of 128000 f32, n = 8: 107 us with 64, 121 with 256;
// 700 rows, bf16: 34 with 64, 33 with 256.
template <int NT>
constexpr int lp_occ() { return NT == 256 ? 3 : (NT == 64 ? 12 : 16); }  // CTAs of an SM
template <int NT>
constexpr int lp_ring() { return NT == 32 ? 12 : 8; }  // 16-byte loads a thread has in flight or at hand
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

// 2^a within 2 units in the last place (the special-function unit's; 2^-22 of each term, as much as
// the rounding of its argument). expf would take the kernel's issue slots, its bound for many rows.
PI_DEV float ex2(float a) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a));
    return r;
}
// x - m for x <= m, held above -200 (e^-200 is 0 in f32), so that a masked value (-inf or
// the type's lowest) adds 0 to both sums instead of 0 * inf; NaN stays NaN.
PI_DEV float lp_shift(float x, float m) { return max_nan(x - m, -200.0f); }

template <int N>
PI_DEV float lp_max(const float* f) {
    float a = fmaxf(f[0], f[1]), b = fmaxf(f[2], f[3]);
    if constexpr (N == 8) {
        a = fmaxf(a, fmaxf(f[4], f[5]));
        b = fmaxf(b, fmaxf(f[6], f[7]));
    }
    return fmaxf(a, b);
}

// Largest of the warp's values, NaN dropped.
PI_DEV float warp_max(float v) {
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
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

// Keeps the n best of the cnt keys in buf, in order, P a lane; the n-th one's value (-inf where
// there are fewer). A function of its own: it is rare, and the loop around it is to stay in
// the instruction cache.
template <int P>
__device__ __noinline__ float lp_keep_best(uint64_t* buf, int cnt, int n, int lane) {
    uint64_t k[P];
#pragma unroll
    for (int i = 0; i < P; ++i) k[i] = lane + 32 * i < cnt ? buf[lane + 32 * i] : 0;
    __syncwarp();
    const int keep = min(n, cnt);
    uint64_t best = 0;
#pragma unroll 1
    for (int r = 0; r < keep; ++r) {
        uint64_t mine = 0;
#pragma unroll
        for (int i = 0; i < P; ++i) mine = k[i] > mine ? k[i] : mine;
        best = warp_max_key(mine);
#pragma unroll
        for (int i = 0; i < P; ++i) k[i] = k[i] == best ? 0 : k[i];  // keys are distinct
        if (lane == 0) buf[r] = best;
    }
    __syncwarp();
    return keep == n ? lp_key_value(best) : -INFINITY;
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

    PI_DEV void compact() {
        const float least = cnt <= 64 ? lp_keep_best<2>(buf, cnt, n, lane) : lp_keep_best<CAP / 32>(buf, cnt, n, lane);
        if (cnt >= n) {
            thr = fmaxf(thr, least);
            incl = false;
        }
        cnt = min(cnt, n);
    }
    PI_DEV bool passes(float x) const { return x > thr || (incl && x == thr); }
    // N values per lane, index i0 + j, once more in memory at `at`; every lane calls it
    template <int N, typename ET>
    PI_DEV void add(const float* x, float vmax, const ET* at, uint32_t i0) {
        if (!__any_sync(0xffffffffu, passes(vmax))) return;
        if (cnt + 32 * N > CAP) compact();
        uint32_t mask = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) mask |= (uint32_t)passes(x[j]) << j;
        while (true) {  // one value of every lane that has any, mostly a single time
            const uint32_t b = __ballot_sync(0xffffffffu, mask != 0);
            if (!b) break;
            if (mask) {
                const int j = __ffs(mask) - 1;
                buf[cnt + __popc(b & ((1u << lane) - 1u))] = lp_key(lp_float(at[j]), i0 + j);
                mask &= mask - 1;
            }
            cnt += __popc(b);
        }
        __syncwarp();
        // A threshold that stays behind lets value after value in (32000 values, n = 1, threshold of
        // the first 512: 62 of them, one in most steps): it follows.
        if (n == 1) {
            thr = fmaxf(thr, warp_max(vmax));
            incl = false;
        } else if (cnt >= n + 24) {
            compact();
        }
    }
};

// The n best of `cnt` distinct keys in `all` to best[0..n) (0 where there are fewer): a
// key's place is the number of larger ones, counted by four lanes.
template <int NT>
PI_DEV void lp_rank(const uint64_t* all, int cnt, uint64_t* best, int n, int tid) {
    if (tid < n && tid >= cnt) best[tid] = 0;
    for (int i0 = 0; i0 < cnt; i0 += NT / 4) {
        const int i = i0 + (tid >> 2);
        const uint64_t k = i < cnt ? all[i] : ~0ull;
        int r = 0;
        for (int j = tid & 3; j < cnt; j += 4) r += all[j] > k;
        r += __shfl_xor_sync(0xffffffffu, r, 1);
        r += __shfl_xor_sync(0xffffffffu, r, 2);
        if (i < cnt && r < n && (tid & 3) == 0) best[r] = k;
    }
}

// The joined state of a warp's lanes (in every lane): the common maximum first, one rescaling,
// then plain sums.
PI_DEV void lp_join_warp(LpStat& st) {
    const float m = warp_max(st.m), dm = lp_shift(st.m, m), e = ex2(dm * LP_LOG2E);
    st.w = warp_sum(fmaf(dm, st.s, st.w) * e);
    st.s = warp_sum(st.s * e);
    st.m = m;
}

// Row blockIdx.x / C, share blockIdx.x % C. The first LP_U loads of a thread give maxima of
// groups: the n-th largest of the warps' (n <= 8) or of 64 groups of four lanes (a warp alone:
// of its lanes) is reached by n values at least, so only what reaches it is kept from the start
// (with 256 threads about n values of the first 4096 or 8192, then n / i of the i-th step), and
// the buffers hardly ever fill.
template <typename ET, bool TOP, int NT>
__global__ __launch_bounds__(NT, lp_occ<NT>()) void k_token_logprobs(const LogprobArgs a) {
    constexpr int LP_NT = NT, LP_W = NT / 32, LP_D = lp_ring<NT>();
    constexpr int GROUP = NT == 32 ? 1 : (NT == 64 ? 2 : 4), GROUPS = NT / GROUP;  // groups of lanes whose maxima give the threshold
    constexpr int KEYS = NT == 256 ? LP_MAXC * LP_MAXTOP : 320;    // keys ranked together; one warp has no cluster
    constexpr int NV = 16 / (int)sizeof(ET);
    constexpr int CAP = 64 + 32 * NV;  // n kept after compact() and one load of every lane
    __shared__ uint64_t s_buf[TOP ? LP_W * CAP : 1];
    __shared__ uint64_t s_all[TOP ? KEYS : 1];
    __shared__ uint64_t s_lists[TOP && NT == 256 ? LP_MAXC * LP_MAXTOP : 1];  // the cluster's lists, in its first CTA
    __shared__ LpStat s_stats[LP_MAXC];                                       // and its states
    __shared__ uint64_t s_best[LP_MAXTOP];
    __shared__ LpStat s_stat[LP_W], s_cta;
    __shared__ float s_max[GROUPS], s_thr;
    __shared__ int s_cnt[LP_W];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int C = NT == 256 ? a.C : 1;
    const int row32 = (int)(blockIdx.x / (unsigned)C), rank = (int)blockIdx.x - row32 * C;
    const int64_t row = row32;
    const ET* x = reinterpret_cast<const ET*>(a.logits) + row * a.ld;
    // values before the first 16-byte boundary and after the last whole 16 bytes are read
    // one by one by the first warp of the row
    const int head = (int)min((int64_t)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(ET)), a.V);
    const int nvec = (int)((a.V - head) / NV), tail = head + nvec * NV;
    const int4* xv = reinterpret_cast<const int4*>(x + head);
    const int step = C * LP_NT;
    // the row's results from its joined state and s_best, by `nthr` threads
    auto answer = [&](const LpStat& t, int i0, int nthr) {
        // s == 0: the row's mask leaves nothing; s NaN: a NaN or +inf, no distribution
        const bool none = t.s == 0.0f, bad = t.s != t.s;
        const float log_s = none ? 0.0f : logf(t.s), nan = __int_as_float(0x7fffffff);
        if (i0 == 0 && a.entropy) a.entropy[row] = none ? 0.0f : (bad ? nan : log_s - t.w / t.s);
        for (int64_t j = i0; j < a.n_targets; j += nthr) {
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
            if (i0 < a.n_top) {
                const uint64_t k = bad ? 0 : s_best[i0];
                a.top_ids[row * a.n_top + i0] = k ? (int32_t)lp_key_index(k) : -1;
                a.top_logp[row * a.n_top + i0] = bad ? nan : (k ? (lp_key_value(k) - t.m) - log_s : -INFINITY);
            }
        }
    };
    const bool edges = rank == 0 && warp == 0;
    // the first CTA of the cluster must run before the others write into its shared memory
    if (NT == 256 && C > 1) cluster_arrive();

    // this thread's maximum and packed sums of e^(x - m) and (x - m) e^(x - m)
    float m = LP_LOWEST;
    uint64_t s2 = 0, w2 = 0;
    auto raise = [&](float to) {
        const float dm = lp_shift(m, to), e = ex2(dm * LP_LOG2E);
        const uint64_t e2 = pack2(e, e);
        w2 = mul2(fma2(pack2(dm, dm), s2, w2), e2);
        s2 = mul2(s2, e2);
        m = to;
    };
    auto pair = [&](float x0, float x1) {
        float2 t = unpack2(add2(pack2(x0, x1), pack2(-m, -m)));
        t.x = max_nan(t.x, -200.0f);
        t.y = max_nan(t.y, -200.0f);
        const uint64_t tt = pack2(t.x, t.y);
        const float2 g = unpack2(mul2(tt, pack2(LP_LOG2E, LP_LOG2E)));
        const uint64_t e = pack2(ex2(g.x), ex2(g.y));
        s2 = add2(s2, e);
        w2 = fma2(tt, e, w2);
    };
    LpTop<CAP> top;
    if constexpr (TOP) {
        top.buf = s_buf + warp * CAP;
        top.n = a.n_top;
        top.lane = lane;
    }
    if (edges) {
        const float v = lane < head ? lp_float(x[lane]) : -INFINITY;
        if (lane < head) {
            if (v > m) raise(v);
            pair(v, -INFINITY);
        }
        if constexpr (TOP) top.template add<1>(&v, v, x + lane, (uint32_t)lane);
    }
    // Loads go through a ring in shared memory, of which a thread reads only what it copied itself
    // (no barrier): 32 KB a CTA in flight. In registers 8 KB were (2048 rows of 32000 bf16: 47
    // us, 2.8 TB/s).
    const int minus_inf = sizeof(ET) == 4 ? (int)0xff800000 : (std::is_same_v<ET, __half> ? (int)0xfc00fc00 : (int)0xff80ff80);
    const int4 none = make_int4(minus_inf, minus_inf, minus_inf, minus_inf);
    extern __shared__ __align__(16) int4 s_ring[];
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(s_ring + tid);
    int v0 = rank * LP_NT + tid, slot = 0;
    auto request = [&](int v, int at) {  // a step's loads, one group
#pragma unroll
        for (int u = 0; u < LP_U; ++u)
            if (v + u * step < nvec)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ring + (at + u) * LP_NT * 16),
                             "l"(xv + v + u * step)
                             : "memory");
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < LP_D; i += LP_U) request(v0 + i * step, i);
    bool first = true;
    for (; v0 - tid < nvec || first; v0 += LP_U * step) {
        float f[LP_U][NV], mx = -INFINITY;
        asm volatile("cp.async.wait_group %0;" ::"n"(LP_D / LP_U - 1) : "memory");
#pragma unroll
        for (int u = 0; u < LP_U; ++u) {
            lp_unpack<ET>(v0 + u * step < nvec ? s_ring[(slot + u) * LP_NT + tid] : none, f[u]);  // behind the end: -inf
            mx = fmaxf(mx, lp_max<NV>(f[u]));
        }
        if constexpr (TOP) {
            if (first) {
                if (a.n_top <= LP_W) {
                    const float w = warp_max(mx);
                    if (lane == 0) s_max[warp] = w;
                    __syncthreads();
                    const float mine = s_max[lane % LP_W];
                    int r = 0;
#pragma unroll
                    for (int o = 0; o < LP_W; ++o) r += s_max[o] > mine || (s_max[o] == mine && o < lane % LP_W);
                    const uint32_t b = __ballot_sync(0xffffffffu, r == a.n_top - 1);
                    top.thr = __shfl_sync(0xffffffffu, mine, __ffs(b) - 1);
                } else {
                    float w = mx;
#pragma unroll
                    for (int o = 1; o < GROUP; o <<= 1) w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, o));
                    if (tid % GROUP == 0) s_max[tid / GROUP] = w;
                    __syncthreads();
                    const int i = tid / GROUP;  // the lanes of a group count the maxima above theirs
                    const float mine = s_max[i];
                    int r = 0;
#pragma unroll
                    for (int j = 0; j < GROUPS / GROUP; ++j) {
                        const int o = tid % GROUP + GROUP * j;
                        r += s_max[o] > mine || (s_max[o] == mine && o < i);
                    }
#pragma unroll
                    for (int o = 1; o < GROUP; o <<= 1) r += __shfl_xor_sync(0xffffffffu, r, o);
                    if (r == a.n_top - 1) s_thr = mine;
                    __syncthreads();
                    top.thr = s_thr;
                }
                top.incl = top.thr > -INFINITY;
            }
        }
        if (mx > m) raise(mx);
#pragma unroll
        for (int u = 0; u < LP_U; ++u)
#pragma unroll
            for (int j = 0; j < NV; j += 2) pair(f[u][j], f[u][j + 1]);
        if constexpr (TOP) {
            if (__any_sync(0xffffffffu, top.passes(mx)))
// 16-bit types: a loop over values read once more, for the code to fit the instruction cache (600
// rows of 32000 bf16, n = 8: 50 us unrolled, 31 so; f32, half as many values: 90 as a loop, 83)
#pragma unroll (NV == 4 ? LP_U : 1)
                for (int u = 0; u < LP_U; ++u) {
                    const int4* at = &s_ring[(slot + u) * LP_NT + tid];
                    const uint32_t i0 = (uint32_t)head + (uint32_t)(v0 + u * step) * NV;  // behind the end: past 2^31
                    if constexpr (NV == 4) {
                        top.template add<NV>(f[u], lp_max<NV>(f[u]), reinterpret_cast<const ET*>(at), i0);
                    } else {
                        float e[NV];
                        lp_unpack<ET>(v0 + u * step < nvec ? *at : none, e);
                        top.template add<NV>(e, lp_max<NV>(e), reinterpret_cast<const ET*>(at), i0);
                    }
                }
            top.incl = false;
        }
        request(v0 + LP_D * step, slot);
        slot = slot + LP_U == LP_D ? 0 : slot + LP_U;
        first = false;
    }
    if (edges) {
        const bool in = lane < (int)(a.V - tail);  // tail + lane may pass 2^31
        const float v = in ? lp_float(x[(int64_t)tail + lane]) : -INFINITY;
        if (in) {
            if (v > m) raise(v);
            pair(v, -INFINITY);
        }
        if constexpr (TOP) top.template add<1>(&v, v, x + (int64_t)tail + lane, (uint32_t)tail + lane);
    }

    const float2 ss = unpack2(s2), ww = unpack2(w2);
    LpStat st{m, ss.x + ss.y, ww.x + ww.y};
    // join: lanes, warps, then the CTAs of the cluster
    lp_join_warp(st);
    if (lane == 0) s_stat[warp] = st;
    if constexpr (TOP) {
        if (lane == 0) s_cnt[warp] = top.cnt;
        __syncthreads();
        int at = 0, total = 0;
        for (int i = 0; i < LP_W; ++i) {
            if (i < warp) at += s_cnt[i];
            total += s_cnt[i];
        }
        if (NT > 32 && total > 256) {
            __syncthreads();
            if (top.cnt > a.n_top) top.compact();
            if (lane == 0) s_cnt[warp] = top.cnt;
            __syncthreads();
            at = total = 0;
            for (int i = 0; i < LP_W; ++i) {
                if (i < warp) at += s_cnt[i];
                total += s_cnt[i];
            }
        }
        for (int i = lane; i < top.cnt; i += 32) s_all[at + i] = top.buf[i];
        __syncthreads();
        if ((NT < 256 || C == 1) && total <= 32) {  // few keys: the first warp ranks them, the others are done
            if (warp != 0) return;
            const uint64_t k = lane < total ? s_all[lane] : 0;
            int r = 0;
            for (int j = 0; j < total; ++j) r += s_all[j] > k;
            if (lane < a.n_top) s_best[lane] = 0;
            __syncwarp();
            if (lane < total && r < a.n_top) s_best[r] = k;
            __syncwarp();
            LpStat t = s_stat[lane % LP_W];
            if (lane >= LP_W) t.s = t.w = 0.0f;
            lp_join_warp(t);
            answer(t, lane, 32);
            return;
        }
        lp_rank<NT>(s_all, total, s_best, a.n_top, tid);
    } else {
        __syncthreads();
        if (C == 1) {
            if (warp != 0) return;
            LpStat t = s_stat[lane % LP_W];
            if (lane >= LP_W) t.s = t.w = 0.0f;
            lp_join_warp(t);
            answer(t, lane, 32);
            return;
        }
    }
    if (warp == 0) {
        LpStat t = s_stat[lane % LP_W];
        if (lane >= LP_W) t.s = t.w = 0.0f;
        lp_join_warp(t);
        if (lane == 0) s_cta = t;
    }
    if (NT == 256 && C > 1) {
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
            if (lane >= C) t.s = t.w = 0.0f;
            lp_join_warp(t);
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
            lp_rank<NT>(s_all, s_cnt[0], s_best, a.n_top, tid);
        }
    }
    __syncthreads();
    answer(s_cta, tid, LP_NT);
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

template <typename ET, int NT>
cudaError_t launch_logprobs(pi_ctx* ctx, const LogprobArgs& a, cudaStream_t st) {
    auto kern = a.n_top > 0 ? k_token_logprobs<ET, true, NT> : k_token_logprobs<ET, false, NT>;
    if (a.C > 8)
        if (cudaError_t e = allow_wide_cluster((const void*)kern, ctx->device)) return e;
    // always raised: static and dynamic shared memory together pass the default of 48 KB
    pi_smem_attr((const void*)kern, 64 * 1024);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.T * a.C));
    cfg.blockDim = dim3(NT);
    cfg.dynamicSmemBytes = lp_ring<NT>() * NT * 16;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)a.C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = a.C > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, a);
}
template <typename ET>
cudaError_t launch_rows(pi_ctx* ctx, const LogprobArgs& a, int threads, cudaStream_t st) {
    return threads == 32   ? launch_logprobs<ET, 32>(ctx, a, st)
           : threads == 64 ? launch_logprobs<ET, 64>(ctx, a, st)
                           : launch_logprobs<ET, 256>(ctx, a, st);
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
    const int64_t nvec = V * es / 16, sms = ctx->sm_count > 0 ? ctx->sm_count : 148;
    // with 256 threads a row, as many CTAs to it as still run all at once with two loads a thread each
    const int threads = T >= 8 * sms ? 32 : (T >= 5 * sms ? 64 : 256);
    if (threads == 256)
        while (a.C < LP_MAXC && T * a.C * 2 <= lp_occ<256>() * sms && nvec >= (int64_t)a.C * 2 * 2 * 256) a.C *= 2;
    PiProfScope ps(ctx, st, "k_token_logprobs");
    const cudaError_t e = dtype == PI_QT_F32   ? launch_rows<float>(ctx, a, threads, st)
                          : dtype == PI_QT_F16 ? launch_rows<__half>(ctx, a, threads, st)
                                               : launch_rows<__nv_bfloat16>(ctx, a, threads, st);
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
