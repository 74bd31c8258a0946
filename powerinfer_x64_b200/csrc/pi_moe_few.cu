// The whole MoE layer of a few tokens (at most 16) in two kernels, Q4_0 experts
// (model/mod.rs:1239-1571; the decode chain of pi_moe.cu takes 7-8 launches):
//
//   k_few_logits   RMSNorm (optional) and the router's exact logits
//   k_few_experts  top-k and gates, gate/up and SwiGLU, a barrier of the grid, down, the
//                  gate-weighted sum, the gated shared expert and the residual
//
// Routing keeps the reference's arithmetic bit for bit (sequential f32 logits, its softmax,
// ties to the lowest index), so the experts and gates are those of pi_moe_route. Expert
// products are f32 sums of f32 activations and the exact nibble values, one multiply by
// the block's scale per 32 terms (the reference dequantises and sums sequentially,
// quant/mod.rs:958-969): equal to f32 rounding, as on the layer's other Q4_0 paths.
//
// Bound: the bytes of the experts that the tokens use, and for one token the latency of the
// chain: the sequential logit (about 4.2 cycles an input), two launches, the barrier and
// three dependent trips to memory. k_few_experts is launched cooperatively: its barrier
// needs every CTA resident, also while another stream runs the same.
#include "pi_common.cuh"
#include "pi_internal.h"
#include "pi_topk.cuh"

#include <algorithm>
#include <exception>

namespace {

constexpr int FEW_T = 16;  // tokens at most

// ---------------------------------------------------------------------------
// k_few_logits: CTA = two router rows (row E: the shared expert's gate) and a group of
// tokens, all in shared memory (row pitch d + 4 floats: a lane's 16-byte reads of its own
// row fall into distinct banks). Four lanes per token run the reference's four sums of
// squares, then one lane per (row, token) its sequential logit.
// ---------------------------------------------------------------------------
constexpr int FL_T = 128, FL_R = 2;

struct FewLogitArgs {
    const float *x, *router, *bias;
    int T, d, E, group, norm;  // group: tokens of a CTA
    float *normed, *logits;
    uint32_t* bar;
};

__global__ __launch_bounds__(FL_T) void k_few_logits(const FewLogitArgs a) {
    pdl_wait();
    extern __shared__ __align__(16) float s_rows[];
    __shared__ float s_inv[FEW_T];
    const int tid = threadIdx.x, d = a.d, pitch = d + 4;
    const int e0 = blockIdx.x * FL_R, nrow = min(FL_R, a.E + 1 - e0);
    const int t0 = blockIdx.y * a.group, nt = min(a.group, a.T - t0);
    float *s_w = s_rows, *s_x = s_rows + FL_R * pitch;
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) *a.bar = 0;  // of the next kernel
    for (int i = tid; i < (nrow + nt) * (d / 4); i += FL_T) {
        const int r = i / (d / 4), c = i - r * (d / 4);
        const float* src = r < nrow ? a.router + (int64_t)(e0 + r) * d : a.x + (int64_t)(t0 + r - nrow) * d;
        float* dst = r < nrow ? s_w + r * pitch : s_x + (r - nrow) * pitch;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst + 4 * c)),
                     "l"(src + 4 * c)
                     : "memory");
    }
    asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    if (a.norm) {
        // ss = (l0 + l1) + (l2 + l3) over elements 4m + lane, x * (1 / sqrt(ss / d + eps))
        // (simd.rs:116-137, ops.rs:13-27)
        if (tid < 4 * FEW_T) {
            const int t = tid >> 2, l = tid & 3;
            float acc = 0.0f;
            if (t < nt) {
                const float* r = s_x + t * pitch + l;
#pragma unroll 16
                for (int j = 0; j < d; j += 4) acc = fadd(acc, fmul(r[j], r[j]));
            }
            const float a1 = __shfl_down_sync(0xffffffffu, acc, 1);
            const float a2 = __shfl_down_sync(0xffffffffu, acc, 2);
            const float a3 = __shfl_down_sync(0xffffffffu, acc, 3);
            if (l == 0) {
                const float ss = fadd(fadd(acc, a1), fadd(a2, a3));
                s_inv[t] = fdiv(1.0f, __fsqrt_rn(fadd(fdiv(ss, (float)d), 1e-6f)));
            }
        }
        __syncthreads();
        for (int i = tid; i < nt * (d / 4); i += FL_T) {
            const int t = i / (d / 4), c = i - t * (d / 4);
            float4 v = *reinterpret_cast<const float4*>(s_x + t * pitch + 4 * c);
            const float inv = s_inv[t];
            v = make_float4(fmul(v.x, inv), fmul(v.y, inv), fmul(v.z, inv), fmul(v.w, inv));
            *reinterpret_cast<float4*>(s_x + t * pitch + 4 * c) = v;
            if (blockIdx.x == 0) *reinterpret_cast<float4*>(a.normed + (int64_t)(t0 + t) * d + 4 * c) = v;
        }
        __syncthreads();
    }
    const int r = tid % FL_R, t = tid / FL_R;
    if (r >= nrow || t >= nt) return;
    const float *wr = s_w + r * pitch, *xr = s_x + t * pitch;
    float acc = 0.0f;
#pragma unroll 32
    for (int i = 0; i < d; i += 4) {
        const float4 w = *reinterpret_cast<const float4*>(wr + i);
        const float4 v = *reinterpret_cast<const float4*>(xr + i);
        acc = fadd(acc, fmul(w.x, v.x));
        acc = fadd(acc, fmul(w.y, v.y));
        acc = fadd(acc, fmul(w.z, v.z));
        acc = fadd(acc, fmul(w.w, v.w));
    }
    if (a.bias && e0 + r < a.E) acc = fadd(acc, a.bias[e0 + r]);
    a.logits[(int64_t)(t0 + t) * (a.E + 1) + e0 + r] = acc;
}

// ---------------------------------------------------------------------------
// k_few_experts
// ---------------------------------------------------------------------------
constexpr int FE_T = 512, FE_W = FE_T / 32;
constexpr int FE_TB = 4;         // tokens that share a decoded weight
constexpr int FE_PART = 512;     // (column group, expert) sums of a CTA kept at a time
constexpr int FE_MAXU = 513;     // used experts and the shared one

struct FewExpertArgs {
    const uint8_t *g, *u, *dn, *gs, *us, *dns;       // routed and shared nibbles
    const __half *gd, *ud, *dd, *gsd, *usd, *dsd;    // their block scales
    const float *x, *xin, *logits;                   // x: the residual; xin: the (normed) input
    int T, d, f, E, k, has_shared, has_shgate, residual;
    int group, n_groups;  // tokens whose inputs a CTA keeps for gate/up; such groups
    float *h, *out;       // h [T][k + shared][f]
    uint32_t *bar, *err;
};

// Eight nibbles of a word (element 2i low, 2i + 1 high in byte i) as pairs of f32: a byte
// put below 0x4B000000 is the float 2^23 + n, from which 2^23 + 8 is taken exactly.
PI_DEV void nibble_pairs(uint32_t w, uint64_t* v) {
    const uint32_t lo = w & 0x0F0F0F0Fu, hi = (w >> 4) & 0x0F0F0F0Fu;
    const uint64_t off = pack2(-8388616.0f, -8388616.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = add2(pack2(__uint_as_float(__byte_perm(lo, 0x4B000000u, 0x7440 + i)),
                          __uint_as_float(__byte_perm(hi, 0x4B000000u, 0x7440 + i))),
                    off);
}
PI_DEV uint32_t word_of(const int4& v, int i) {
    return (uint32_t)(i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w)));
}

// Gate and up of two neighbouring rows for TB tokens: lane l holds blocks l + 32 c of each row.
// xs[t]: the token's inputs in shared memory, 36 floats a block (lanes' 16-byte reads then
// fall into distinct banks). sum[2 row + (0 gate, 1 up)][token], over all lanes.
template <int CPL, int TB>
PI_DEV void gateup_rows(const uint8_t* G, const uint8_t* U, const __half* GD, const __half* UD, int d,
                        const float* const (&xs)[TB], int lane, float (&sum)[4][TB]) {
    int4 w[2][4];
    float s[2][4];
    const int nb = d / 32;
    auto load = [&](int c, int4 (&q)[4], float (&sc)[4]) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int64_t b = (int64_t)r * nb + lane + 32 * c;
            q[2 * r] = ld_stream(G + b * 16);
            q[2 * r + 1] = ld_stream(U + b * 16);
            sc[2 * r] = __half2float(GD[b]);
            sc[2 * r + 1] = __half2float(UD[b]);
        }
    };
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int t = 0; t < TB; ++t) sum[v][t] = 0.0f;
    load(0, w[0], s[0]);
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
        if (c + 1 < CPL) load(c + 1, w[(c + 1) & 1], s[(c + 1) & 1]);
        uint64_t part[4][TB];
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
            for (int t = 0; t < TB; ++t) part[v][t] = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {  // words: eight elements
            uint64_t n[4][4];
#pragma unroll
            for (int v = 0; v < 4; ++v) nibble_pairs(word_of(w[c & 1][v], q), n[v]);
#pragma unroll
            for (int t = 0; t < TB; ++t) {
                const ulonglong2* xp = reinterpret_cast<const ulonglong2*>(xs[t] + (lane + 32 * c) * 36 + q * 8);
                const ulonglong2 x0 = xp[0], x1 = xp[1];
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    part[v][t] = fma2(n[v][0], x0.x, part[v][t]);
                    part[v][t] = fma2(n[v][1], x0.y, part[v][t]);
                    part[v][t] = fma2(n[v][2], x1.x, part[v][t]);
                    part[v][t] = fma2(n[v][3], x1.y, part[v][t]);
                }
            }
        }
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
            for (int t = 0; t < TB; ++t) {
                const float2 p = unpack2(part[v][t]);
                sum[v][t] = fmaf(s[c & 1][v], p.x + p.y, sum[v][t]);
            }
    }
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int t = 0; t < TB; ++t) sum[v][t] = warp_sum(sum[v][t]);
}

// One expert's part of eight output columns (rows of D, lane-tiled by quarters of a row):
// lane 4 r + q sums quarter q of row r; returns the row's sum in its lanes. hq: h in shared
// memory, quarter q at q (8 BPQ * 4 + 4) floats.
template <int BPQ>
PI_DEV float down_rows(const uint8_t* D, const __half* DD, const float* hs, int lane) {
    const int r = lane >> 2, q = lane & 3;
    int4 w[BPQ];
    float s[BPQ];
#pragma unroll
    for (int b = 0; b < BPQ; ++b) {
        w[b] = ld_stream(D + (b * 32 + lane) * 16);
        s[b] = __half2float(DD[(r * 4 + q) * BPQ + b]);
    }
    const float* hp = hs + q * (BPQ * 32 + 4);
    float sum = 0.0f;
#pragma unroll
    for (int b = 0; b < BPQ; ++b) {
        uint64_t part = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint64_t n[4];
            nibble_pairs(word_of(w[b], i), n);
            const ulonglong2* x = reinterpret_cast<const ulonglong2*>(hp + b * 32 + i * 8);
            const ulonglong2 x0 = x[0], x1 = x[1];
            part = fma2(n[0], x0.x, part);
            part = fma2(n[1], x0.y, part);
            part = fma2(n[2], x1.x, part);
            part = fma2(n[3], x1.y, part);
        }
        const float2 p = unpack2(part);
        sum = fmaf(s[b], p.x + p.y, sum);
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    return sum;
}

// Barrier of a cooperatively launched grid, used once: *bar counts up from 0. The wait is
// bounded (2^24 polls, the later ones 32 ns apart: about half a second); when it runs out
// the kernel records PI_DEVERR_TIMEOUT and the CTA returns.
PI_DEV bool grid_barrier(uint32_t* bar, uint32_t* err, int* s_ok) {
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        atomicAdd(bar, 1u);
        int ok = 0;
        for (uint32_t it = 0; it < (1u << 24); ++it) {
            uint32_t v;
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(bar) : "memory");
            if (v >= gridDim.x) {
                ok = 1;
                break;
            }
            if (it > 4096) __nanosleep(32);
        }
        if (!ok) atomicOr(err, PI_DEVERR_TIMEOUT);
        *s_ok = ok;
    }
    __syncthreads();
    return *s_ok != 0;
}

template <int CPL, int NPL>
__global__ __launch_bounds__(FE_T, 1) void k_few_experts(const FewExpertArgs a) {
    extern __shared__ __align__(16) float s_dyn[];  // gate/up: inputs of the group's tokens, then top-k scratch; down: h
    __shared__ int s_idx[FEW_T * 32], s_sel[FE_W][32], s_use[FE_MAXU], s_mask[FE_MAXU], s_nuse, s_ok;
    __shared__ float s_gate[FEW_T * 32], s_share[FEW_T], s_part[FE_PART * 8];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int T = a.T, d = a.d, f = a.f, E = a.E, k = a.k, nb = d / 32, slots = k + a.has_shared;
    const int grp = blockIdx.x % a.n_groups, t0 = grp * a.group, nt = min(a.group, T - t0);
    const int cta = blockIdx.x / a.n_groups, n_cta = (gridDim.x - grp + a.n_groups - 1) / a.n_groups;

    // the group's inputs, 36 floats a block
    for (int i = tid; i < nt * (d / 4); i += FE_T) {
        const int t = i / (d / 4), c = i - t * (d / 4);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(
                         s_dyn + (t * nb + (c >> 3)) * 36 + (c & 7) * 4)),
                     "l"(a.xin + (int64_t)(t0 + t) * d + 4 * c)
                     : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    // routing of every token (a warp each), in every CTA
    if (warp < T)
        topk_token<NPL>(a.logits, warp, E, k, a.has_shgate, s_idx, s_gate, s_share, nullptr,
                        s_dyn + a.group * nb * 36 + warp * 32 * NPL, s_sel[warp], lane);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    // the experts that the group's tokens use, ascending, with the tokens of each
    for (int e = tid; e < E; e += FE_T) s_mask[e] = 0;
    __syncthreads();
    for (int i = tid; i < nt * k; i += FE_T) atomicOr(&s_mask[s_idx[t0 * k + i]], 1 << (i / k));
    __syncthreads();
    if (warp == 0) {
        int n = 0;
        for (int e0 = 0; e0 < E; e0 += 32) {
            const int m = e0 + lane < E ? s_mask[e0 + lane] : 0;
            const uint32_t b = __ballot_sync(0xffffffffu, m != 0);
            if (m) s_use[n + __popc(b & ((1u << lane) - 1u))] = e0 + lane;
            n += __popc(b);
        }
        if (a.has_shared && lane == 0) {
            s_use[n] = E;
            s_mask[E] = (1 << nt) - 1;
        }
        if (lane == 0) s_nuse = n + a.has_shared;
    }
    __syncthreads();

    // gate, up and SwiGLU: a warp takes two rows of an expert for all of its tokens
    const int half_f = f / 2, n_unit = s_nuse * half_f;
    for (int unit = cta * FE_W + warp; unit < n_unit; unit += n_cta * FE_W) {
        const int e = s_use[unit / half_f], row = 2 * (unit % half_f);
        const bool sh = e == E;
        uint32_t mask = s_mask[e];
        const int64_t r = (sh ? 0 : (int64_t)e * f) + row;
        const uint8_t *G = (sh ? a.gs : a.g) + r * (d / 2), *U = (sh ? a.us : a.u) + r * (d / 2);
        const __half *GD = (sh ? a.gsd : a.gd) + r * nb, *UD = (sh ? a.usd : a.ud) + r * nb;
        auto store = [&](int t, const float (&g)[2], const float (&u)[2]) {  // lanes 0, 1: a row each
            int j = k;
            if (!sh) j = __ffs(__ballot_sync(0xffffffffu, lane < k && s_idx[(t0 + t) * k + lane] == e)) - 1;
            if (lane < 2)
                a.h[((int64_t)(t0 + t) * slots + j) * f + row + lane] =
                    swiglu_ref(lane ? g[1] : g[0], lane ? u[1] : u[0]);
        };
        if (__popc(mask) == 1) {
            const int t = __ffs(mask) - 1;
            const float* xs[1] = {s_dyn + t * nb * 36};
            float sum[4][1];
            gateup_rows<CPL, 1>(G, U, GD, UD, d, xs, lane, sum);
            const float g[2] = {sum[0][0], sum[2][0]}, u[2] = {sum[1][0], sum[3][0]};
            store(t, g, u);
        } else {
            while (mask) {
                int tok[FE_TB], n = 0;
                const float* xs[FE_TB];
#pragma unroll
                for (int i = 0; i < FE_TB; ++i) {  // a batch that is not full repeats its last token
                    if (mask) {
                        tok[i] = __ffs(mask) - 1;
                        mask &= mask - 1;
                        ++n;
                    } else {
                        tok[i] = tok[i > 0 ? i - 1 : 0];
                    }
                    xs[i] = s_dyn + tok[i] * nb * 36;
                }
                float sum[4][FE_TB];
                gateup_rows<CPL, FE_TB>(G, U, GD, UD, d, xs, lane, sum);
#pragma unroll
                for (int i = 0; i < FE_TB; ++i) {
                    if (i >= n) break;
                    const float g[2] = {sum[0][i], sum[2][i]}, u[2] = {sum[1][i], sum[3][i]};
                    store(tok[i], g, u);
                }
            }
        }
    }
    if (!grid_barrier(a.bar, a.err, &s_ok)) return;

    // down: the CTA's share of the (token, eight columns) units, token by token
    const int per_tok = d / 8, bpq = f / 128, hp = f + 16;  // hp: floats of a padded h row
    const int64_t all = (int64_t)T * per_tok;
    const int ub = (int)(all * blockIdx.x / gridDim.x), ue = (int)(all * (blockIdx.x + 1) / gridDim.x);
    for (int u = ub; u < ue;) {
        const int t = u / per_tok, tok_end = min(ue, (t + 1) * per_tok);
        __syncthreads();
        for (int i = tid; i < slots * (f / 4); i += FE_T) {
            const int j = i / (f / 4), c = 4 * (i - j * (f / 4)), q = c / (f / 4);
            *reinterpret_cast<float4*>(s_dyn + j * hp + c + 4 * q) =
                __ldcg(reinterpret_cast<const float4*>(a.h + ((int64_t)t * slots + j) * f + c));
        }
        __syncthreads();
        while (u < tok_end) {
            const int n = min(FE_PART / slots, tok_end - u), col0 = (u - t * per_tok) * 8;
            for (int i = warp; i < n * slots; i += FE_W) {
                const int v = i / slots, j = i - v * slots;
                const int e = j < k ? s_idx[t * k + j] : E;
                const int64_t row = (e == E ? 0 : (int64_t)e * d) + col0 + v * 8;
                const uint8_t* D = (e == E ? a.dns : a.dn) + row * (f / 2);
                const __half* DD = (e == E ? a.dsd : a.dd) + row * (f / 32);
                const float* hs = s_dyn + j * hp;
                float s;
                switch (bpq) {
                    case 1: s = down_rows<1>(D, DD, hs, lane); break;
                    case 2: s = down_rows<2>(D, DD, hs, lane); break;
                    case 4: s = down_rows<4>(D, DD, hs, lane); break;
                    default: s = down_rows<8>(D, DD, hs, lane); break;
                }
                if ((lane & 3) == 0) s_part[(v * slots + j) * 8 + (lane >> 2)] = s;
            }
            __syncthreads();
            for (int i = tid; i < n * 8; i += FE_T) {  // model/mod.rs:1525-1534, :1627-1633
                const float* p = s_part + (i >> 3) * slots * 8 + (i & 7);
                float acc = 0.0f;
                for (int j = 0; j < k; ++j) acc = fadd(acc, fmul(s_gate[t * k + j], p[j * 8]));
                if (a.has_shared) acc = fadd(acc, fmul(s_share[t], p[k * 8]));
                const int64_t o = (int64_t)t * d + col0 + i;
                a.out[o] = a.residual ? fadd(a.x[o], acc) : acc;
            }
            __syncthreads();
            u += n;
        }
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
constexpr size_t FEW_X_BYTES = 152 * 1024;  // inputs of the tokens a CTA keeps for gate/up

struct FewBufs {
    float *logits, *normed, *h;
    uint32_t* bar;
    size_t bytes;
};
FewBufs few_carve(const pi_moe_layer* L, int64_t T, char* base) {
    PiBump b{base};
    FewBufs o;
    o.bar = b.take<uint32_t>(1);
    o.logits = b.take<float>(T * (L->E + 1));
    o.normed = b.take<float>(T * L->d);
    o.h = b.take<float>(T * (L->k + (L->has_shared ? 1 : 0)) * L->f);
    o.bytes = b.off + 256;
    return o;
}

template <int CPL, int NPL>
cudaError_t launch_experts(const FewExpertArgs& a, int sms, cudaStream_t st) {
    const size_t x = (size_t)a.group * (a.d / 32) * 36 * 4, p = (size_t)FE_W * 32 * NPL * 4;
    const size_t h = (size_t)(a.k + a.has_shared) * (a.f + 16) * 4, smem = std::max(x + p, h);
    auto kern = k_few_experts<CPL, NPL>;
    // the limit is always raised: beside the kernel's 26 KB of static shared memory the default
    // of 48 KB would not hold what pi_smem_attr lets pass as small
    pi_smem_attr((const void*)kern, std::max<size_t>(smem, 64 * 1024));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)sms);
    cfg.blockDim = dim3(FE_T);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeCooperative;
    at[0].val.cooperative = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

int few_forward(pi_ctx* ctx, const pi_moe_layer* L, const float* x, int64_t T, float* out, int flags, void* workspace,
                uint64_t workspace_bytes, cudaStream_t st) {
    if (L->ctx->device != ctx->device) return pi_set_error(ctx, PI_ERR_ARG, "moe fused: made on another device");
    if (flags & ~(PI_FWD_RMSNORM | PI_FWD_RESIDUAL))
        return pi_set_error(ctx, PI_ERR_ARG, "moe fused: flags are PI_FWD_RMSNORM and PI_FWD_RESIDUAL");
    if (L->qtype != PI_QT_Q4_0 || L->n_exp != L->E)
        return pi_set_error(ctx, PI_ERR_ARG, "moe fused: a Q4_0 layer that holds all its experts");
    if (T < 0 || T > FEW_T) return pi_set_error(ctx, PI_ERR_ARG, "moe fused: at most 16 tokens");
    if (T == 0) return PI_OK;
    if (!x || !out) return pi_set_error(ctx, PI_ERR_ARG, "moe fused: null pointer");
    if ((((uintptr_t)x | (uintptr_t)out) & 15) || ((uintptr_t)workspace & 255))
        return pi_set_error(ctx, PI_ERR_ARG, "moe fused: x and out 16-byte, the workspace 256-byte aligned");
    const size_t need = few_carve(L, T, nullptr).bytes;
    if (workspace && workspace_bytes < need) return pi_set_error(ctx, PI_ERR_SHORT, "moe fused: workspace too small");
    PiDeviceGuard dev(ctx->device);
    char* scr = (char*)workspace;
    if (!workspace)
        if (int rc = pi_scratch(ctx, st, need, &scr)) return rc;
    const FewBufs B = few_carve(L, T, scr);
    const int d = (int)L->d, E = L->E;
    const bool norm = flags & PI_FWD_RMSNORM;
    {
        PiProfScope ps(ctx, st, "k_few_logits");
        // tokens of a CTA: what 128 KB of shared memory hold
        const int group = (int)std::min<int64_t>(T, (128 * 1024) / (4 * d));
        const size_t smem = sizeof(float) * (size_t)(FL_R + group) * (d + 4);
        pi_smem_attr((const void*)k_few_logits, smem);
        const FewLogitArgs a{x, L->router, L->bias, (int)T, d, E, group, norm ? 1 : 0, B.normed, B.logits, B.bar};
        pi_pdl_launch(k_few_logits, dim3((unsigned)((E + FL_R) / FL_R), (unsigned)((T + group - 1) / group)),
                      dim3(FL_T), smem, st, a);
        if (int rc = pi_cuda_check(ctx, cudaGetLastError(), "moe fused logits")) return rc;
    }
    PiProfScope ps(ctx, st, "k_few_experts");
    const int group = (int)std::min<int64_t>(T, (int64_t)(FEW_X_BYTES / (d / 32 * 36 * 4)));
    FewExpertArgs a = {};
    a.g = (const uint8_t*)L->gate.q;
    a.u = (const uint8_t*)L->up.q;
    a.dn = (const uint8_t*)L->down.q;
    a.gd = L->gate.d;
    a.ud = L->up.d;
    a.dd = L->down.d;
    if (L->has_shared) {
        a.gs = (const uint8_t*)L->gate_sh.q;
        a.us = (const uint8_t*)L->up_sh.q;
        a.dns = (const uint8_t*)L->down_sh.q;
        a.gsd = L->gate_sh.d;
        a.usd = L->up_sh.d;
        a.dsd = L->down_sh.d;
    }
    a.x = x;
    a.xin = norm ? B.normed : x;
    a.logits = B.logits;
    a.T = (int)T;
    a.d = d;
    a.f = (int)L->f;
    a.E = E;
    a.k = L->k;
    a.has_shared = L->has_shared ? 1 : 0;
    a.has_shgate = L->has_shared_gate ? 1 : 0;
    a.residual = flags & PI_FWD_RESIDUAL ? 1 : 0;
    a.group = group;
    a.n_groups = (int)((T + group - 1) / group);
    a.h = B.h;
    a.out = out;
    a.bar = B.bar;
    a.err = ctx->dev_err;
    const int sms = ctx->sm_count > 0 ? ctx->sm_count : 148;
    const bool wide = E > 256;
    cudaError_t e;
    switch (d / 1024) {
        case 1: e = wide ? launch_experts<1, 16>(a, sms, st) : launch_experts<1, 8>(a, sms, st); break;
        case 2: e = wide ? launch_experts<2, 16>(a, sms, st) : launch_experts<2, 8>(a, sms, st); break;
        default: e = wide ? launch_experts<4, 16>(a, sms, st) : launch_experts<4, 8>(a, sms, st); break;
    }
    return pi_cuda_check(ctx, e, "moe fused experts");
}

}  // namespace

extern "C" uint64_t pi_moe_fused_workspace(const pi_moe_layer* L, int64_t T) {
    return L && T > 0 && T <= FEW_T ? few_carve(L, T, nullptr).bytes : 0;
}

extern "C" int pi_moe_forward_fused(pi_ctx* ctx, const pi_moe_layer* L, const float* x, int64_t T, float* out,
                                    int32_t flags, void* workspace, uint64_t workspace_bytes, void* stream) {
    if (!ctx || !L) return PI_ERR_ARG;
    try {
        return few_forward(ctx, L, x, T, out, flags, workspace, workspace_bytes, (cudaStream_t)stream);
    } catch (const std::exception&) {  // an allocation of the host failed
        return PI_ERR_OOM;
    }
}
