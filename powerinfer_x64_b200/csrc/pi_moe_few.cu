// The whole MoE layer of a few tokens (at most 16) in two kernels, Q4_0 experts
// (model/mod.rs:1239-1571; the decode chain of pi_moe.cu takes 7-8 launches):
//
//   k_few_logits   RMSNorm (optional), the router's logits and a bound of their distance from
//                  the reference's
//   k_few_experts  top-k and gates, gate/up and SwiGLU, a barrier of the grid, down, the
//                  gate-weighted sum, the gated shared expert and the residual
//
// The experts chosen are the reference's, bit for bit. Its logits are sequential f32 sums
// (quant/mod.rs:921-935), about 4.2 dependent cycles an input: 5.5 us of a token's 29 at
// n_embd 2048. Here a logit is summed in 32 segments side by side with a bound of how far
// the sequential sum can be from it, and a choice that the bounds leave open (0.4% of
// tokens for normal inputs, and exact ties) is made again from sequential logits, which the
// whole grid makes at the price of one more barrier, and the reference's own softmax and top-k
// (pi_topk.cuh).
//
// Expert products: the reference dequantises Q4_0 rows and sums f32 products (quant/mod.rs:
// 958-969). Here 32 inputs that share a weight scale become fixed-point numbers of 22 bits
// below their largest, held as three int8 terms, so a block's dot with the nibbles is three
// exact integer dots (dp4a: 1.1 instructions a weight and token, against 2.4 for decoding
// nibbles to f32), and one f32 multiply-add per block follows. Values that stand far above the
// rest of their block are held apart in f32 and multiplied one by one: every other value is then
// within 2^-22 of one that four of its 32 reach a 32nd of, so within 2^-17 of the block's
// fourth largest, and an outlier whose weight is 0 costs its neighbours nothing.
//
// Bound: the bytes of the experts that the tokens use; for a token or two the latency of the
// chain (two launches, the barrier and four dependent trips to memory). k_few_experts is launched cooperatively: its
// barrier needs every CTA resident, also while another stream runs the same.
#include "pi_common.cuh"
#include "pi_internal.h"
#include "pi_topk.cuh"

#include <algorithm>
#include <exception>
#include <type_traits>

namespace {

constexpr int FEW_T = 16;  // tokens at most

// ---------------------------------------------------------------------------
// Fixed-point blocks. 32 values in eight lanes, four each: with 2^e the power of two that
// brings the largest of those not held apart into [2^21, 2^22), X = rint(x 2^e) = 65536 q1 + 256
// q2 + q3, each q an int8. A block is 28 words: [term][word of eight elements][even elements, odd
// elements], as the nibbles of a Q4_0 word fall apart (low: even, high: odd), then the scale
// 2^-e / 16 (nibbles come shifted by four bits), then the mask of the values held apart (X = 0
// there), then padding that keeps the lanes' 16-byte reads of neighbouring blocks in distinct
// banks.
//
// Held apart are NaN, infinities, and the largest values as long as fewer than four of the 32
// (of those that are left) reach a 32nd of the largest: none among normal values, some in one of
// 10000 blocks of h (a product of two), one or two in a block with an activation of a hundred times
// its neighbours' size, and all where fewer than four are not 0 or 2^e would pass its range (below
// 2^-99).
// ---------------------------------------------------------------------------
constexpr int FX_WORDS = 28, FX_SCALE = 24, FX_APART = 25;

// Which of a lane's four values of a block are held apart, and the largest magnitude of the block's
// others. All 32 lanes call it, for one odd block among theirs: rare.
__device__ __noinline__ uint2 hold_apart(float4 v) {
    float e[4] = {v.x, v.y, v.z, v.w}, m = 0.0f;
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (!(fabsf(e[i]) < INFINITY)) {
            mine |= 1u << i;
            e[i] = 0.0f;
        }
        m = fmaxf(m, fabsf(e[i]));
    }
    while (true) {
        int n = 0;
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float lim = m * 0x1p-5f;
#pragma unroll
        for (int i = 0; i < 4; ++i) n += fabsf(e[i]) >= lim;
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
        const bool part = m > 0.0f && (n < 4 || m < 0x1p-99f);
        if (!__any_sync(0xffffffffu, part)) return make_uint2(mine, __float_as_uint(m));
        if (part) {
            m = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (fabsf(e[i]) > 0.0f && fabsf(e[i]) >= lim) {
                    mine |= 1u << i;
                    e[i] = 0.0f;
                }
                m = fmaxf(m, fabsf(e[i]));
            }
        }
    }
}

// v: this lane's elements 4j..4j+3 of a block, j = lane % 8; all 32 lanes call it. The lane's
// values are stored at `apart` too where one of them is held apart (null: they are kept elsewhere).
// Returns the block's mask.
PI_DEV uint32_t fix_block(const float4 v, uint32_t* blk, int j, bool store, float* apart) {
    const float own = max_nan(max_nan(fabsf(v.x), fabsf(v.y)), max_nan(fabsf(v.z), fabsf(v.w)));
    float m = own, e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    // a block is as most are where four of its lanes reach the limit
    const uint32_t reach = __ballot_sync(0xffffffffu, own >= m * 0x1p-5f) >> (threadIdx.x & 24);
    uint32_t mine = 0, all = 0;
    if (__any_sync(0xffffffffu, !(m < INFINITY) || (m > 0.0f && (m < 0x1p-99f || __popc(reach & 255u) < 4)))) {
        const uint2 r = hold_apart(v);
        mine = r.x;
        m = __uint_as_float(r.y);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if ((mine >> i) & 1) e[i] = 0.0f;
        all = mine << (4 * j);
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) all |= __shfl_xor_sync(0xffffffffu, all, o);
    }
    const int ex = m > 0.0f ? 21 - ilogbf(m) : 0;
    const float s = ldexpf(1.0f, ex);
    uint32_t even[3] = {0, 0, 0}, odd[3] = {0, 0, 0};  // two bytes of each term
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int X = __float2int_rn(e[i] * s);
        const int q3 = (int)(int8_t)X, X2 = (X - q3) >> 8, q2 = (int)(int8_t)X2, q1 = (X2 - q2) >> 8;
        uint32_t* to = i & 1 ? odd : even;
        to[0] |= (uint32_t)(q1 & 255) << (8 * (i >> 1));
        to[1] |= (uint32_t)(q2 & 255) << (8 * (i >> 1));
        to[2] |= (uint32_t)(q3 & 255) << (8 * (i >> 1));
    }
    if (!store) return 0;
    if (apart && mine) *reinterpret_cast<float4*>(apart) = v;
    uint16_t* h = reinterpret_cast<uint16_t*>(blk);
#pragma unroll
    for (int t = 0; t < 3; ++t) {
        h[t * 16 + (j >> 1) * 4 + (j & 1)] = (uint16_t)even[t];
        h[t * 16 + (j >> 1) * 4 + 2 + (j & 1)] = (uint16_t)odd[t];
    }
    if (j == 0) *reinterpret_cast<uint2*>(blk + FX_SCALE) = make_uint2(__float_as_uint(ldexpf(0.0625f, -ex)), all);
    return all;
}

// Element i of a Q4_0 block of bytes at q, times the block's scale.
PI_DEV float nib_value(const uint8_t* q, int i, __half d) {
    return __half2float(d) * (float)(((__ldg(q + (i >> 1)) >> (4 * (i & 1))) & 15) - 8);
}

// nibbles of a word as 16 (n - 8) in int8: even elements, odd elements
PI_DEV uint32_t nib_even(uint32_t w) { return ((w << 4) & 0xF0F0F0F0u) ^ 0x80808080u; }
PI_DEV uint32_t nib_odd(uint32_t w) { return (w & 0xF0F0F0F0u) ^ 0x80808080u; }
// the value of a block's three dots
PI_DEV float fix_value(const int (&s)[3]) { return fmaf((float)s[0], 65536.0f, (float)(s[1] * 256 + s[2])); }

// ---------------------------------------------------------------------------
// k_few_logits: CTA = R router rows (row E: the shared expert's gate) and a group of tokens in
// shared memory, each row as 32 segments of S = d / 32 floats at a pitch of S + 4 (lanes'
// 16-byte reads of their own segments then fall into distinct banks). A warp takes a (row,
// token), lane l its segment l.
//
// Distance from the reference (u = 2^-24). A sequential sum rounds each product, u |p_i|, and
// each partial sum, u |P_i|; the lanes' sums here do no worse, and joining 32 of them adds 5 u
// sum |p|. With P_start the sum before a lane's segment and L the sum of the absolute partial
// sums inside it, sum |P_i| <= B = sum over lanes of S |P_start| + L; errors of errors are
// below d u < 2.5e-4 of that. So |reference - here| <= u (2.2 B + 12 A + 4 (|l| + |bias|)), A =
// sum |p|, which leaves 3 u A for the normed inputs' own roundings. RMSNorm itself scales
// all inputs of a token alike: the reference's sum of squares, d / 4 sequential additions
// in four lanes, moves a logit by at most (d / 8 + 4) u |l|, this one's, d / 32 fused steps and a
// join of five, by (d / 64 + 5) u |l|: 72 u and d / 8 u at n_embd 4096, held as 96.
// ---------------------------------------------------------------------------
constexpr int FL_T = 256, FL_W = FL_T / 32;
constexpr int FL_GROUP = 4;               // tokens of a CTA
constexpr size_t FL_SMEM = 190 * 1024;

struct FewLogitArgs {
    const float *x, *router, *bias;
    int T, d, E, R, norm;
    float *logits, *eps;  // [T][E + 1], eps: the bounds
    uint32_t *xfix, *bar;  // xfix [T][d / 32][FX_WORDS]: the (normed) inputs in fixed point
    float* xap;            // [T][d]: those held apart, nothing elsewhere
};

__global__ __launch_bounds__(FL_T) void k_few_logits(const FewLogitArgs a) {
    extern __shared__ __align__(16) float s_rows[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int d = a.d, S = d / 32, pitch = 32 * (S + 4), s4 = S / 4;  // s4 = 8, 16 or 32
    const int e0 = blockIdx.x * a.R, nrow = min(a.R, a.E + 1 - e0);
    const int t0 = blockIdx.y * FL_GROUP, nt = min(FL_GROUP, a.T - t0);
    float *s_x = s_rows, *s_w = s_rows + FL_GROUP * pitch;
    auto fetch = [&](float* dst, const float* src, int rows) {
        const int per = d / 4, lg = 31 - __clz(s4);
        for (int i = tid; i < rows * per; i += FL_T) {
            const int r = i / per, c = i - r * per;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(
                             dst + r * pitch + (c >> lg) * (S + 4) + (c & (s4 - 1)) * 4)),
                         "l"(src + (int64_t)r * d + 4 * c)
                         : "memory");
        }
    };
    fetch(s_w, a.router + (int64_t)e0 * d, nrow);  // constant weights: before the wait
    pdl_wait();
    fetch(s_x, a.x + (int64_t)t0 * d, nt);
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid < 2) a.bar[tid] = 0;  // of the next kernel
    asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    if (a.norm) {
        if (warp < nt) {  // x * (1 / sqrt(mean square + eps)), ops.rs:13-27
            float* r = s_x + warp * pitch + lane * (S + 4);
            float ss = 0.0f;
            for (int i = 0; i < S; i += 4) {
                const float4 v = *reinterpret_cast<const float4*>(r + i);
                ss = fmaf(v.x, v.x, fmaf(v.y, v.y, fmaf(v.z, v.z, fmaf(v.w, v.w, ss))));
            }
            const float inv = fdiv(1.0f, __fsqrt_rn(fadd(fdiv(warp_sum(ss), (float)d), 1e-6f)));
            for (int i = 0; i < S; i += 4) {
                float4 v = *reinterpret_cast<const float4*>(r + i);
                v = make_float4(fmul(v.x, inv), fmul(v.y, inv), fmul(v.z, inv), fmul(v.w, inv));
                *reinterpret_cast<float4*>(r + i) = v;
            }
        }
        __syncthreads();
    }
    // the blocks of the group's inputs are shared out over the CTAs of the group
    for (int q0 = 0; q0 * (int)gridDim.x < nt * (d / 32); q0 += FL_T / 8) {
        const int o = (q0 + (tid >> 3)) * gridDim.x + blockIdx.x, j = tid & 7;
        const bool in = o < nt * (d / 32);
        const int t = in ? o / (d / 32) : 0, b = in ? o - t * (d / 32) : 0, i = b * 32 + 4 * j;
        const float4 v = *reinterpret_cast<const float4*>(s_x + t * pitch + (i / S) * (S + 4) + (i & (S - 1)));
        fix_block(v, a.xfix + ((int64_t)(t0 + t) * (d / 32) + b) * FX_WORDS, j, in,
                  a.xap + (int64_t)(t0 + t) * d + i);
    }
    for (int q = warp; q < nrow * nt; q += FL_W) {
        const int r = q / nt, t = q - r * nt, e = e0 + r;
        const float *wr = s_w + r * pitch + lane * (S + 4), *xr = s_x + t * pitch + lane * (S + 4);
        float sum = 0.0f, part = 0.0f, terms = 0.0f;
#pragma unroll 8
        for (int i = 0; i < S; i += 4) {
            const float4 w = *reinterpret_cast<const float4*>(wr + i);
            const float4 v = *reinterpret_cast<const float4*>(xr + i);
            const float p[4] = {w.x * v.x, w.y * v.y, w.z * v.z, w.w * v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sum = fadd(sum, p[j]);
                part += fabsf(sum);
                terms += fabsf(p[j]);
            }
        }
        float upto = sum;  // sum of this and the earlier segments
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const float v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        float before = __shfl_up_sync(0xffffffffu, upto, 1);
        if (lane == 0) before = 0.0f;
        const float B = warp_sum(fmaf((float)S, fabsf(before), part)), A = warp_sum(terms);
        const float l = __shfl_sync(0xffffffffu, upto, 31);
        if (lane == 0) {
            const float b = a.bias && e < a.E ? a.bias[e] : 0.0f;
            float bound = 2.2f * B + 12.0f * A + 4.0f * fabsf(l);
            if (a.norm) bound += ((float)d * 0.125f + 96.0f) * fabsf(l);
            // exact: nothing but zeros to add (products that vanish here and, other norms, not in the
            // reference are below 2^-148 and move no probability), or a masked expert
            const bool exact = A == 0.0f || (b == -INFINITY && bound < INFINITY);
            a.logits[(int64_t)(t0 + t) * (a.E + 1) + e] = l + b;
            a.eps[(int64_t)(t0 + t) * (a.E + 1) + e] = exact ? 0.0f : (bound + 4.0f * fabsf(b)) * 5.9604645e-8f;
        }
    }
}

// ---------------------------------------------------------------------------
// k_few_experts
// ---------------------------------------------------------------------------
constexpr int FE_T = 512, FE_W = FE_T / 32;
constexpr int FE_TB = 4;         // tokens at most that share a decoded weight
constexpr int FE_SLOTS = 33;     // experts of a token and the shared one at most
constexpr int FE_PART = 512;     // (column group, expert) sums of a CTA kept at a time
constexpr int FE_MAXE = 513;     // experts and the shared one (a layer has 512 at most, a thread each)
constexpr int FE_ITEMS = FE_MAXE + FEW_T / FE_TB;

struct FewExpertArgs {
    const uint8_t *g, *u, *dn, *gs, *us, *dns;       // routed and shared nibbles
    const __half *gd, *ud, *dd, *gsd, *usd, *dsd;    // their block scales
    const float* x;                                  // the layer's input
    const uint32_t* xfix;
    const float* xap;
    const float *logits, *eps, *router, *bias;
    int T, d, f, E, k, has_shared, has_shgate, norm, residual;
    int group, n_groups;  // tokens whose inputs a CTA keeps for gate/up; such groups
    float *exact;         // [T][E + 1], of tokens that the bounds leave open
    float *h, *out;       // h [T][k + shared][f]
    uint32_t *bar, *err;
};

PI_DEV uint32_t word_of(const int4& v, int i) {
    return (uint32_t)(i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w)));
}

// Gate and up of two neighbouring rows: where they start, and one chunk (the lane's block
// l + 32 c of each row) in registers.
struct RowPtrs {
    const uint8_t *g, *u;
    const __half *gd, *ud;
};
struct RowChunk {
    int4 w[4];  // row 0 gate, up, row 1 gate, up
    __half s[4];
    PI_DEV void load(const RowPtrs& p, int nb, int blk) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int b = r * nb + blk;
            w[2 * r] = ld_stream(p.g + b * 16);
            w[2 * r + 1] = ld_stream(p.u + b * 16);
            s[2 * r] = p.gd[b];
            s[2 * r + 1] = p.ud[b];
        }
    }
};

// sum[v][t] += row-vector v of the chunk times token t's block (xs[t]: the token's fixed-point
// blocks in shared memory).
template <int TB>
PI_DEV void chunk_products(const RowChunk& k, const uint32_t* const (&xs)[TB], int blk, float (&sum)[4][TB]) {
    int dot[4][TB][3];
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int t = 0; t < TB; ++t) dot[v][t][0] = dot[v][t][1] = dot[v][t][2] = 0;
#pragma unroll
    for (int q = 0; q < 2; ++q) {  // two words, sixteen elements
        uint32_t n[4][4];
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t x = word_of(k.w[v], 2 * q + i);
                n[v][2 * i] = nib_even(x);
                n[v][2 * i + 1] = nib_odd(x);
            }
#pragma unroll
        for (int t = 0; t < TB; ++t)
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                const int4 x = *reinterpret_cast<const int4*>(xs[t] + blk * FX_WORDS + p * 8 + q * 4);
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    int& o = dot[v][t][p];
                    o = dp4a((int)n[v][0], x.x, o);
                    o = dp4a((int)n[v][1], x.y, o);
                    o = dp4a((int)n[v][2], x.z, o);
                    o = dp4a((int)n[v][3], x.w, o);
                }
            }
    }
#pragma unroll
    for (int t = 0; t < TB; ++t) {
        const float sx = __uint_as_float(xs[t][blk * FX_WORDS + FX_SCALE]);
#pragma unroll
        for (int v = 0; v < 4; ++v)
            sum[v][t] = fmaf(__half2float(k.s[v]) * sx, fix_value(dot[v][t]), sum[v][t]);
    }
}

// Which inputs of a group's tokens are held apart: a bit for each block that has some, and where they
// are few the list of them, by their place modulo 8 and then in order, each with its value in every
// token (0 where it is not held apart). Outliers mostly stand at the same few places in every token.
constexpr int AP_LIST = 64;
struct ApartInputs {
    uint32_t any, n;  // n > AP_LIST: too many for the list
    uint32_t blk[FEW_T][4];
    uint16_t found[AP_LIST], at[AP_LIST];  // in order; by place modulo 8, whose parts start at first[]
    int first[9];
    float value[FEW_T][AP_LIST];
};

// The list, by the whole CTA; rare.
template <int CPL>
__device__ __noinline__ void list_apart(ApartInputs& s, const uint32_t* s_x, const float* xap, int nt) {
    constexpr int nb = 32 * CPL;
    const int tid = threadIdx.x;
    if (tid < 32) {
        int n = 0;
        for (int c = 0; c < CPL; ++c) {
            uint32_t m = 0;  // of block tid + 32 c in any token
            for (int t = 0; t < nt; ++t) m |= s_x[(t * nb + tid + 32 * c) * FX_WORDS + FX_APART];
            int upto = __popc(m);
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (tid >= o) upto += v;
            }
            for (int i = n + upto - __popc(m); m; m &= m - 1, ++i)
                if (i < AP_LIST) s.found[i] = (uint16_t)((tid + 32 * c) * 32 + __ffs(m) - 1);
            n += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (tid == 0) s.n = n;
        __syncwarp();
        if (tid < 9 && n <= AP_LIST) {
            int pos = 0;
            for (int i = 0; i < n; ++i) pos += (s.found[i] & 7) < tid;
            s.first[tid] = pos;
            for (int i = 0; i < n; ++i)
                if ((s.found[i] & 7) == tid) s.at[pos++] = s.found[i];
        }
    }
    __syncthreads();
    if (s.n <= AP_LIST)
        for (int i = tid; i < nt * AP_LIST; i += FE_T) {
            const int t = i / AP_LIST, q = i % AP_LIST;
            float v = 0.0f;
            if (q < s.n && (s_x[(t * nb + (s.at[q] >> 5)) * FX_WORDS + FX_APART] >> (s.at[q] & 31)) & 1)
                v = xap[t * nb * 32 + s.at[q]];
            s.value[t][q] = v;
        }
    __syncthreads();
}

// c[t] += this lane's part of what the values held apart add to row-vector lane / 8 of an item's unit
// (rows row, row + 1 of expert e) for its tokens, numbered in the bytes of toks within the CTA's
// group: of all elements those at lane % 8 modulo 8, in order, whichever tokens stand beside one another (so
// a token's sums are the same alone). The weights, read a moment ago, come from L2. A function of its own: it is rare, and the loop around it has
// no registers to spare.
template <int CPL>
__device__ __noinline__ float4 apart_products(const FewExpertArgs& a, const ApartInputs& s, const uint32_t* s_x, int t0,
                                              uint32_t toks, int e, int row, float4 c, int lane) {
    constexpr int d = 1024 * CPL, nb = d / 32;
    const bool up = lane & 8, sh = e == a.E;
    const int64_t r = (sh ? 0 : (int64_t)e * a.f) + row + (lane >> 4);
    const uint8_t* w = (up ? (sh ? a.us : a.u) : (sh ? a.gs : a.g)) + r * (d / 2);
    const __half* sc = (up ? (sh ? a.usd : a.ud) : (sh ? a.gsd : a.gd)) + r * nb;
    const int tok[FE_TB] = {(int)(toks & 255), (int)(toks >> 8 & 255), (int)(toks >> 16 & 255), (int)(toks >> 24)};
    float sum[FE_TB] = {c.x, c.y, c.z, c.w};
    if (s.n <= AP_LIST) {
#pragma unroll 2
        for (int q = s.first[lane & 7]; q < s.first[(lane & 7) + 1]; ++q) {
            const int at = s.at[q];
            const float v = nib_value(w + (at >> 5) * 16, at & 31, sc[at >> 5]);
#pragma unroll
            for (int t = 0; t < FE_TB; ++t) sum[t] = fmaf(v, s.value[tok[t]][q], sum[t]);
        }
        return make_float4(sum[0], sum[1], sum[2], sum[3]);
    }
    for (int q = 0; q < CPL; ++q) {
        uint32_t blks = 0;
#pragma unroll
        for (int t = 0; t < FE_TB; ++t) blks |= s.blk[tok[t]][q];
        for (; blks; blks &= blks - 1) {
            const int b = 32 * q + __ffs(blks) - 1;
            uint32_t mask[FE_TB], any = 0;
#pragma unroll
            for (int t = 0; t < FE_TB; ++t) {
                mask[t] = s_x[(tok[t] * nb + b) * FX_WORDS + FX_APART] >> (lane & 7);
                any |= mask[t];
            }
            for (int i = 0; i < 32; i += 8) {
                if (!((any >> i) & 1)) continue;
                const float v = nib_value(w + b * 16, i + (lane & 7), sc[b]);
#pragma unroll
                for (int t = 0; t < FE_TB; ++t)
                    if ((mask[t] >> i) & 1)
                        sum[t] = fmaf(v, a.xap[(int64_t)(t0 + tok[t]) * d + b * 32 + i + (lane & 7)], sum[t]);
            }
        }
    }
    return make_float4(sum[0], sum[1], sum[2], sum[3]);
}

// All chunks of a unit for TB tokens, the unit's first chunk being in `k`; leaves there the first
// chunk of the next unit (at `next`), which is on its way while the last one is worked on.
// out[t]: eight parts of each row's sum, in lanes 0-7 those of the first row's gate, 8-15 of its up, 16-23
// of the second row's gate, 24-31 of its up.
template <int CPL, int TB>
PI_DEV void gateup_rows(RowChunk& k, const RowPtrs& at, const RowPtrs& next, const uint32_t* const (&xs)[TB],
                        int lane, float* out) {
    constexpr int nb = 32 * CPL;
    RowChunk other;
    float sum[4][TB];
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int t = 0; t < TB; ++t) sum[v][t] = 0.0f;
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
        RowChunk &now = c & 1 ? other : k, &then = c & 1 ? k : other;
        if (c + 1 < CPL) then.load(at, nb, lane + 32 * (c + 1));
        else then.load(next, nb, lane);
        chunk_products<TB>(now, xs, lane + 32 * c, sum);
    }
    if (CPL & 1) k = other;
    // sums over the lanes, four at once: after two halvings lane l has row-vector l / 8's part
#pragma unroll
    for (int t = 0; t < TB; ++t) {
        const bool hi = lane & 16, mid = lane & 8;
        float a = hi ? sum[2][t] : sum[0][t], b = hi ? sum[3][t] : sum[1][t];
        a += __shfl_xor_sync(0xffffffffu, hi ? sum[0][t] : sum[2][t], 16);
        b += __shfl_xor_sync(0xffffffffu, hi ? sum[1][t] : sum[3][t], 16);
        out[t] = (mid ? b : a) + __shfl_xor_sync(0xffffffffu, mid ? a : b, 8);
    }
}

// h of one expert in shared memory: BPQ fixed-point blocks per quarter of a row, the quarters
// apart so that the four lanes of a row read distinct banks.
PI_DEV int h_quarter(int bpq) { return bpq * FX_WORDS + (bpq == 1 ? 0 : 4); }

// One expert's part of eight output columns (rows of D, lane-tiled by quarters of a row): the
// lane's blocks in registers, and their sum. Lane 4 r + q sums quarter q of row r; the row's
// sum is returned in its lanes.
template <int BPQ>
struct DownRows {
    int4 w[BPQ];
    __half s[BPQ];
    PI_DEV void load(const uint8_t* D, const __half* DD, int lane) {
#pragma unroll
        for (int b = 0; b < BPQ; ++b) {
            w[b] = ld_stream(D + (b * 32 + lane) * 16);
            s[b] = DD[lane * BPQ + b];
        }
    }
    PI_DEV float sum(const uint32_t* hs, int lane) const {
        const uint32_t* hp = hs + (lane & 3) * h_quarter(BPQ);
        float sum = 0.0f;
#pragma unroll
        for (int b = 0; b < BPQ; ++b) {
            int dot[3] = {0, 0, 0};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t w0 = word_of(w[b], 2 * i), w1 = word_of(w[b], 2 * i + 1);
                const uint32_t n[4] = {nib_even(w0), nib_odd(w0), nib_even(w1), nib_odd(w1)};
#pragma unroll
                for (int p = 0; p < 3; ++p) {
                    const int4 x = *reinterpret_cast<const int4*>(hp + b * FX_WORDS + p * 8 + i * 4);
                    dot[p] = dp4a((int)n[0], x.x, dot[p]);
                    dot[p] = dp4a((int)n[1], x.y, dot[p]);
                    dot[p] = dp4a((int)n[2], x.z, dot[p]);
                    dot[p] = dp4a((int)n[3], x.w, dot[p]);
                }
            }
            sum = fmaf(__half2float(s[b]) * __uint_as_float(hp[b * FX_WORDS + FX_SCALE]), fix_value(dot), sum);
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        return sum;
    }
};
// Adds what the values of h held apart give to the sums of a pass, part[unit][expert][column] of n units of
// eight columns from col0 on: blks[expert] has a bit for each block that has some, s_h is the
// fixed-point h and h its f32 values. By the whole CTA; rare.
template <int BPQ>
__device__ __noinline__ void apart_down(const FewExpertArgs& a, const int* idx, const uint32_t* blks, const uint32_t* s_h,
                                        const float* h, int n, int col0, float* part) {
    constexpr int f = 128 * BPQ, hp = 4 * BPQ * FX_WORDS + (BPQ == 1 ? 0 : 16);
    const int slots = a.k + a.has_shared;
    for (int i = threadIdx.x; i < n * slots * 8; i += FE_T) {
        const int v = i / (8 * slots), j = (i >> 3) - v * slots;
        const bool sh = j == a.k;
        const int64_t row = (sh ? 0 : (int64_t)idx[j] * a.d) + col0 + 8 * v;  // eight rows are tiled together
        const uint8_t* D = (sh ? a.dns : a.dn) + row * (f / 2);
        const __half* DD = (sh ? a.dsd : a.dd) + row * (f / 32);
        float s = 0.0f;
        for (uint32_t m = blks[j]; m; m &= m - 1) {
            const int q = (__ffs(m) - 1) / BPQ, b = (__ffs(m) - 1) % BPQ, lane = 4 * (i & 7) + q;
            for (uint32_t e = s_h[j * hp + q * h_quarter(BPQ) + b * FX_WORDS + FX_APART]; e; e &= e - 1)
                s = fmaf(nib_value(D + (b * 32 + lane) * 16, __ffs(e) - 1, DD[lane * BPQ + b]),
                         __ldcg(h + j * f + (q * BPQ + b) * 32 + __ffs(e) - 1), s);
        }
        part[i] += s;
    }
    __syncthreads();
}

// Barrier of a cooperatively launched grid, each used once: *bar counts up from 0. The wait
// ends after 2^31 cycles of the SM (1.1 s at 1.965 GHz), whatever a poll takes: the kernel then
// records PI_DEVERR_TIMEOUT and the CTA returns.
PI_DEV bool grid_barrier(uint32_t* bar, uint32_t* err, int* s_ok) {
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        atomicAdd(bar, 1u);
        int ok = 0;
        long long start = 0;
        for (uint32_t it = 0;; ++it) {
            uint32_t v;
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(bar) : "memory");
            if (v >= gridDim.x) {
                ok = 1;
                break;
            }
            if (it > 4096) __nanosleep(32);
            if ((it & 255) == 255) {
                const long long now = clock64();
                if (it == 255) start = now;
                else if (now - start > (1ll << 31)) break;
            }
        }
        if (!ok) atomicOr(err, PI_DEVERR_TIMEOUT);
        *s_ok = ok;
    }
    __syncthreads();
    return *s_ok != 0;
}

// Top-k and gates of one token from logits and their bounds, by one warp; false where the
// bounds leave the reference's choice open. The reference ranks rounded probabilities
// (model/mod.rs:1278-1303): logits apart by 2^-16 (1 + their distance from the largest) have
// distinct ones as long as none underflows. So the choice is certain where the selected stand
// that far above the others; or where some of both tie exactly (a row of zeros, which pads a
// batch), the lowest indexes among those being the selected ones, and the rest stand that far
// above or below them. A logit of -inf with a bound of 0 is a masked expert. Gates are
// renormalised over the selected, so the softmax's full sum cancels.
template <int NPL>
PI_DEV bool topk_certain(const float* logits, const float* eps, int E, int k, int has_shgate, int32_t* idx,
                         float* gates, float* share, int lane) {
    float l[NPL], hi[NPL];
    uint32_t key[NPL];
    float m = -INFINITY;
    bool known = true;
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const int e = lane + 32 * j;
        l[j] = e < E ? __ldcg(logits + e) : -INFINITY;
        const float ep = e < E ? __ldcg(eps + e) : 0.0f;
        hi[j] = l[j] + ep;  // l itself where the bound is 0, above it otherwise
        known = known && ((fabsf(l[j]) < INFINITY && ep < INFINITY) || (l[j] == -INFINITY && ep == 0.0f));
        const uint32_t b = __float_as_uint(l[j] + 0.0f);  // -0 as 0
        key[j] = e < E ? ((b & 0x80000000u) ? ~b : (b | 0x80000000u)) : 0u;
        m = fmaxf(m, l[j]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (!__all_sync(0xffffffffu, known)) return false;
    int mine = 0x7fffffff;  // lane r: the r-th selected expert, its logit and that one's lower end
    float lm = 0.0f, low = INFINITY;
    for (int r = 0; r < k; ++r) {
        uint32_t mk = 0;
#pragma unroll
        for (int j = 0; j < NPL; ++j) mk = max(mk, key[j]);
        mk = __reduce_max_sync(0xffffffffu, mk);
        uint32_t me = 0xffffffffu;
#pragma unroll
        for (int j = NPL - 1; j >= 0; --j)
            if (key[j] == mk) me = lane + 32 * j;
        const int e = (int)__reduce_min_sync(0xffffffffu, me);
        float lo = INFINITY;
        if ((e & 31) == lane) {
#pragma unroll
            for (int j = 0; j < NPL; ++j)
                if (j == (e >> 5)) {
                    key[j] = 0;
                    lo = l[j] > -INFINITY ? 2.0f * l[j] - hi[j] : -INFINITY;
                    hi[j] = -INFINITY;
                }
        }
        lo = __shfl_sync(0xffffffffu, lo, e & 31);
        if (lane == r) {
            mine = e;
            lm = __uint_as_float((mk & 0x80000000u) ? (mk ^ 0x80000000u) : ~mk);
            low = lo;
        }
    }
    const float v = __shfl_sync(0xffffffffu, lm, k - 1);  // the last selected
    bool tie = false;
    float high = -INFINITY;  // upper end of those not selected, but for those that tie with v
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const bool same = hi[j] == v && l[j] == v;
        tie = tie || same;
        high = fmaxf(high, same ? -INFINITY : hi[j]);
    }
    tie = __any_sync(0xffffffffu, tie) && __shfl_sync(0xffffffffu, low, k - 1) == v;
    if (!tie)
#pragma unroll
        for (int j = 0; j < NPL; ++j) high = fmaxf(high, hi[j]);
    if (tie && low == v && lm == v) low = INFINITY;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    }
    const float edge = tie ? v : low, apart = 0x1p-16f * (1.0f + (m - edge));
    if (!(edge - m > -80.0f) || !(edge > high + apart) || (tie && !(low > v + apart))) return false;
    const float p = lane < k ? expf(lm - m) : 0.0f, sum = warp_sum(p);
    int rank = 0;  // ascending experts, model/mod.rs:1303
    for (int r = 0; r < k; ++r) rank += __shfl_sync(0xffffffffu, mine, r) < mine;
    if (lane < k) {
        idx[rank] = mine;
        gates[rank] = p / sum;
    }
    if (lane == 0) *share = has_shgate ? 1.0f / (1.0f + expf(-__ldcg(logits + E))) : 1.0f;
    return true;
}

// The reference's logits of the tokens in `open`, to a.exact [T][E + 1]: norms (four sequential sums of
// squares, simd.rs:116-137) by a warp a token in every CTA, then sequential chains, a thread for each
// of the CTA's rows and open tokens; the CTAs of the grid share the rows. Both go through
// shared memory (s: FE_PART * 8 floats), in coalesced pieces of which the next is on its way. Only
// for tokens that topk_certain leaves open: 18 us for three of n_embd 2048 and 256 experts, 28 for
// fifteen, 7 of them the norms (each CTA making all chains for itself, token by token: 90 us a token).
constexpr int EX_COLS = 128, EX_PITCH = EX_COLS + 4;
__device__ __noinline__ void exact_logits(const FewExpertArgs& a, uint32_t open, float* s) {
    __shared__ int s_tok[FEW_T];
    __shared__ float s_inv[FEW_T];
    constexpr int ROWS = FE_PART * 8 / EX_PITCH, PER = (ROWS * EX_COLS / 4 + FE_T - 1) / FE_T;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n = __popc(open), d = a.d;
    if (tid < 32 && (open >> tid) & 1) s_tok[__popc(open & ((1u << tid) - 1u))] = tid;
    __syncthreads();
    if (warp < n) {
        float inv = 1.0f;
        if (a.norm) {
            const float* x = a.x + (int64_t)s_tok[warp] * d + lane * 4;
            float *strip = s + warp * 256, acc = 0.0f;
            float4 v = *reinterpret_cast<const float4*>(x), w = *reinterpret_cast<const float4*>(x + 128);
            for (int c = 0; c < d; c += 256) {
                *reinterpret_cast<float4*>(strip + lane * 4) = v;
                *reinterpret_cast<float4*>(strip + 128 + lane * 4) = w;
                __syncwarp();
                if (c + 256 < d) {
                    v = *reinterpret_cast<const float4*>(x + c + 256);
                    w = *reinterpret_cast<const float4*>(x + c + 384);
                }
                if (lane < 4)
#pragma unroll 16
                    for (int j = lane; j < 256; j += 4) acc = fadd(acc, fmul(strip[j], strip[j]));
                __syncwarp();
            }
            const float a1 = __shfl_sync(0xffffffffu, acc, 1), a2 = __shfl_sync(0xffffffffu, acc, 2),
                        a3 = __shfl_sync(0xffffffffu, acc, 3);
            inv = fdiv(1.0f, __fsqrt_rn(fadd(fdiv(fadd(fadd(acc, a1), fadd(a2, a3)), (float)d), 1e-6f)));
        }
        if (lane == 0) s_inv[warp] = inv;
    }
    __syncthreads();
    const int rows = a.E + 1, end = (int)((int64_t)rows * (blockIdx.x + 1) / gridDim.x);
    for (int e0 = (int)((int64_t)rows * blockIdx.x / gridDim.x); e0 < end; e0 += ROWS - n) {
        // a piece: columns of nr router rows, then of the n tokens
        const int nr = min(ROWS - n, end - e0), r = tid / n, i = tid - r * n;
        float4 v[PER];
        auto fetch = [&](int c) {
#pragma unroll
            for (int q = 0; q < PER; ++q) {
                const int at = tid + q * FE_T, row = at / (EX_COLS / 4), col = c + at % (EX_COLS / 4) * 4;
                if (row < nr) v[q] = __ldg(reinterpret_cast<const float4*>(a.router + (int64_t)(e0 + row) * d + col));
                else if (row < nr + n)
                    v[q] = *reinterpret_cast<const float4*>(a.x + (int64_t)s_tok[row - nr] * d + col);
            }
        };
        fetch(0);
        float acc = 0.0f;
        for (int c = 0; c < d; c += EX_COLS) {
#pragma unroll
            for (int q = 0; q < PER; ++q) {
                const int at = tid + q * FE_T, row = at / (EX_COLS / 4), col = at % (EX_COLS / 4) * 4;
                if (row >= nr + n) continue;
                float4 u = v[q];
                if (a.norm && row >= nr) {
                    const float inv = s_inv[row - nr];
                    u = make_float4(fmul(u.x, inv), fmul(u.y, inv), fmul(u.z, inv), fmul(u.w, inv));
                }
                *reinterpret_cast<float4*>(s + row * EX_PITCH + col) = u;
            }
            __syncthreads();
            if (c + EX_COLS < d) fetch(c + EX_COLS);
            if (r < nr) {
                const float *w = s + r * EX_PITCH, *x = s + (nr + i) * EX_PITCH;
#pragma unroll 8
                for (int j = 0; j < EX_COLS; j += 4) {
                    const float4 p = *reinterpret_cast<const float4*>(w + j), u = *reinterpret_cast<const float4*>(x + j);
                    acc = fadd(acc, fmul(p.x, u.x));
                    acc = fadd(acc, fmul(p.y, u.y));
                    acc = fadd(acc, fmul(p.z, u.z));
                    acc = fadd(acc, fmul(p.w, u.w));
                }
            }
            __syncthreads();
        }
        if (r < nr)
            a.exact[(int64_t)s_tok[i] * rows + e0 + r] = a.bias && e0 + r < a.E ? fadd(acc, a.bias[e0 + r]) : acc;
    }
}

struct FewRouting {  // in shared memory: [T][k], [T][k], [T]
    const int* idx;
    const float *gate, *share;
};

// The barrier and what follows it: the CTA's share of the (token, eight columns) units, token by
// token, a warp to each expert's part of a unit. A warp's first weights are in its registers
// before the barrier, each next one's on their way while one is worked on.
template <int BPQ>
PI_DEV void down_phase(const FewExpertArgs& a, const int d, const FewRouting& r, uint32_t* s_h, float* s_part,
                       uint32_t (*s_apart)[FE_SLOTS + 1], int* s_ok) {
    constexpr int f = 128 * BPQ, hp = 4 * BPQ * FX_WORDS + (BPQ == 1 ? 0 : 16);  // hp: words of an expert's h
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int T = a.T, k = a.k, slots = k + a.has_shared, per_tok = d / 8;
    const int64_t all = (int64_t)T * per_tok;
    const int ub = (int)(all * blockIdx.x / gridDim.x), ue = (int)(all * (blockIdx.x + 1) / gridDim.x);
    DownRows<BPQ> cur, nxt;
    // part i of a pass: expert j = i % slots of its unit v = i / slots
    auto load = [&](DownRows<BPQ>& to, int t, int col0, int v, int j) {
        const int c = col0 + v * 8;
        if (j == k) {
            to.load(a.dns + c * (f / 2), a.dsd + c * (f / 32), lane);
        } else {
            const int64_t row = (int64_t)r.idx[t * k + j] * d + c;
            to.load(a.dn + row * (f / 2), a.dd + row * (f / 32), lane);
        }
    };
    const int v0 = warp / slots, j0 = warp - v0 * slots, dv = FE_W / slots, dj = FE_W - dv * slots;
    auto pass = [&](int u) {  // units of one token that are summed together, a thread for each column
        return min(min(FE_PART / slots, FE_T / 8), min(ue, (u / per_tok + 1) * per_tok) - u);
    };
    float residual = 0.0f;
    auto begin = [&](int u) {  // a warp's first weights of the pass from unit u on
        const int t = u / per_tok, n = pass(u);
        if (warp < n * slots) load(cur, t, (u - t * per_tok) * 8, v0, j0);
        if (a.residual && tid < n * 8) residual = a.x[(int64_t)u * 8 + tid];
    };
    if (ub < ue) begin(ub);
    if (tid <= FE_SLOTS) s_apart[0][tid] = 0;
    if (!grid_barrier(a.bar, a.err, s_ok)) return;
    for (int u = ub, tok = -1, turn = 1; u < ue;) {
        const int t = u / per_tok, n = pass(u), col0 = (u - t * per_tok) * 8;
        if (t != tok) {
            const float* ht = a.h + (int64_t)t * slots * f;
            turn ^= 1;  // this token's masks; the next one's are cleared meanwhile
            const int n4 = slots * (f / 4);
            auto fetch = [&](int i0) { return __ldcg(reinterpret_cast<const float4*>(ht) + min(i0 + tid, n4 - 1)); };
            float4 v = fetch(0);
            for (int i0 = 0; i0 < n4; i0 += FE_T) {  // whole warps: eight lanes make a block
                const int i = min(i0 + tid, n4 - 1), j = i / (f / 4), b = (i & (f / 4 - 1)) >> 3;
                const float4 now = v;
                v = fetch(i0 + FE_T);  // on its way meanwhile
                const uint32_t apart = fix_block(now, s_h + j * hp + (b / BPQ) * h_quarter(BPQ) + (b % BPQ) * FX_WORDS,
                                                 i & 7, i0 + tid < n4, nullptr);
                if (apart && (i & 7) == 0) {
                    atomicOr(&s_apart[turn][j], 1u << b);
                    s_apart[turn][FE_SLOTS] = 1;
                }
            }
            if (tid <= FE_SLOTS) s_apart[turn ^ 1][tid] = 0;
            tok = t;
            __syncthreads();
        }
        for (int i = warp, v = v0, j = j0; i < n * slots; i += FE_W) {
            const int now = j;
            v += dv;
            j += dj;
            if (j >= slots) {
                j -= slots;
                ++v;
            }
            if (i + FE_W < n * slots) load(nxt, t, col0, v, j);
            const float s = cur.sum(s_h + now * hp, lane);
            if ((lane & 3) == 0) s_part[i * 8 + (lane >> 2)] = s;
            cur = nxt;
        }
        __syncthreads();
        if (s_apart[turn][FE_SLOTS])
            apart_down<BPQ>(a, r.idx + t * k, s_apart[turn], s_h, a.h + (int64_t)t * slots * f, n, col0, s_part);
        if (tid < n * 8) {  // model/mod.rs:1525-1534, :1627-1633
            const float* p = s_part + (tid >> 3) * slots * 8 + (tid & 7);
            float acc = 0.0f;
            for (int j = 0; j < k; ++j) acc = fadd(acc, fmul(r.gate[t * k + j], p[j * 8]));
            if (a.has_shared) acc = fadd(acc, fmul(r.share[t], p[k * 8]));
            a.out[(int64_t)u * 8 + tid] = a.residual ? fadd(residual, acc) : acc;
        }
        __syncthreads();
        u += n;
        cur = DownRows<BPQ>();  // nothing of it is kept over the rare call above
        if (u < ue) begin(u);
    }
}

template <int CPL, int NPL, int BPQ>
__global__ __launch_bounds__(FE_T, 1) void k_few_experts(const __grid_constant__ FewExpertArgs a) {
    extern __shared__ __align__(16) uint32_t s_dyn[];  // gate/up: inputs of the group's tokens; down: h
    __shared__ int s_idx[FEW_T * 32], s_use[FE_ITEMS], s_mask[FE_T], s_item[FE_ITEMS], s_count[FE_W], s_nuse, s_ok;
    __shared__ ApartInputs s_apart;
    __shared__ uint32_t s_open, s_hblk[2][FE_SLOTS + 1];
    __shared__ __align__(16) float s_part[FE_PART * 8];
    __shared__ float s_gate[FEW_T * 32], s_share[FEW_T];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int d = 1024 * CPL, nb = d / 32, f = 128 * BPQ;
    const int T = a.T, E = a.E, k = a.k, slots = k + a.has_shared;
    const int grp = blockIdx.x % a.n_groups, t0 = grp * a.group, nt = min(a.group, T - t0);
    const int cta = blockIdx.x / a.n_groups, n_cta = (gridDim.x - grp + a.n_groups - 1) / a.n_groups;

    {  // the group's inputs
        const uint32_t to = (uint32_t)__cvta_generic_to_shared(s_dyn);
        const uint32_t* from = a.xfix + (int64_t)t0 * nb * FX_WORDS;
        for (int i = tid; i < nt * nb * (FX_WORDS / 4); i += FE_T)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + i * 16), "l"(from + i * 4) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    // routing of every token (a warp each), in every CTA
    if (tid == 0) s_open = s_apart.any = 0;
    s_mask[tid] = 0;
    __syncthreads();
    if (warp < T &&
        !topk_certain<NPL>(a.logits + (int64_t)warp * (E + 1), a.eps + (int64_t)warp * (E + 1), E, k, a.has_shgate,
                           s_idx + warp * k, s_gate + warp * k, s_share + warp, lane) &&
        lane == 0)
        atomicOr(&s_open, 1u << warp);
    __syncthreads();
    if (const uint32_t open = s_open) {  // the same in every CTA
        exact_logits(a, open, s_part);
        if (!grid_barrier(a.bar + 1, a.err, &s_ok)) return;
        for (int half = 0; half < 2; ++half) {  // s_part: the scratch of eight tokens' top-k
            if (warp / 8 == half && (open >> warp) & 1)
                topk_token<NPL>(a.exact, warp, E, k, a.has_shgate, s_idx, s_gate, s_share, nullptr,
                                s_part + warp % 8 * FE_T, s_item + 32 * warp, lane);
            __syncthreads();
        }
    }
    // The group's work: items of an expert and up to four of its tokens, which share the decoded
    // weights. The shared expert's come first, then those of several tokens, so that the
    // heaviest are spread evenly over the warps. Thread e counts the items of expert e.
    for (int i = tid; i < nt * k; i += FE_T) atomicOr(&s_mask[s_idx[t0 * k + i]], 1 << (i / k));
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    if (warp < nt)  // which blocks of its inputs have values held apart
#pragma unroll
        for (int c = 0; c < CPL; ++c) {
            const uint32_t b =
                __ballot_sync(0xffffffffu, s_dyn[(warp * nb + lane + 32 * c) * FX_WORDS + FX_APART] != 0);
            if (lane == 0) s_apart.blk[warp][c] = b;
            if (lane == 0 && b) s_apart.any = 1;
        }
    {
        const int n_sh = a.has_shared ? (nt + FE_TB - 1) / FE_TB : 0;
        int m = tid < E ? s_mask[tid] : 0;
        const int p = __popc(m), mine = p == 1 ? 1 << 16 : (p + FE_TB - 1) / FE_TB;  // light << 16 | heavy
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        if (lane == 31) s_count[warp] = upto;
        __syncthreads();
        int before = 0, total = 0;
#pragma unroll
        for (int w = 0; w < FE_W; ++w) {
            const int c = s_count[w];
            if (w < warp) before += c;
            total += c;
        }
        before += upto - mine;
        const int heavy = total & 0xffff;
        int at = n_sh + (p == 1 ? heavy + (before >> 16) : (before & 0xffff));
        for (; m; ++at) {
            int take = 0;
            for (int i = 0; i < FE_TB && m; ++i) {
                take |= m & -m;
                m &= m - 1;
            }
            s_use[at] = tid;
            s_item[at] = take;
        }
        if (tid < n_sh) {
            s_use[tid] = E;
            s_item[tid] = ((1 << min(FE_TB, nt - FE_TB * tid)) - 1) << (FE_TB * tid);
        }
        if (tid == 0) s_nuse = n_sh + heavy + (total >> 16);
    }
    __syncthreads();

    // gate, up and SwiGLU: a warp takes two rows of an expert for the tokens of an item
    constexpr int half_f = f / 2;
    const int lf = 31 - __clz(half_f), n_unit = s_nuse * half_f, stride = n_cta * FE_W;
    auto rows = [&](int unit) {
        const int e = s_use[unit >> lf], r = 2 * (unit & (half_f - 1));
        if (e == E)
            return RowPtrs{a.gs + r * (d / 2), a.us + r * (d / 2), a.gsd + r * nb, a.usd + r * nb};
        const int64_t q = (int64_t)(e * f + r);  // E f < 2^20
        return RowPtrs{a.g + q * (d / 2), a.u + q * (d / 2), a.gd + q * nb, a.ud + q * nb};
    };
    auto gate_up = [&](auto any) {
        constexpr bool APART = decltype(any)::value;
        RowChunk chunk;
        RowPtrs at = {}, next = {};
        const int first = cta * FE_W + warp;
        if (first < n_unit) {
            at = rows(first);
            chunk.load(at, nb, lane);
        }
        for (int unit = first; unit < n_unit; unit += stride) {
            const int item = unit >> lf, e = s_use[item], row = 2 * (unit & (half_f - 1));
            uint32_t mask = s_item[item];
            next = unit + stride < n_unit ? rows(unit + stride) : at;  // the last one reads its own first chunk again
            int tok[FE_TB], n = 0;
            const uint32_t* xs[FE_TB];
#pragma unroll
            for (int i = 0; i < FE_TB; ++i) {  // an item that is not full repeats its last token
                if (mask) {
                    tok[i] = __ffs(mask) - 1;
                    mask &= mask - 1;
                    ++n;
                } else {
                    tok[i] = tok[i > 0 ? i - 1 : 0];
                }
                xs[i] = s_dyn + tok[i] * nb * FX_WORDS;
            }
            float sum[FE_TB] = {};
            if (n == 1) {
                const uint32_t* const x1[1] = {xs[0]};
                gateup_rows<CPL, 1>(chunk, at, next, x1, lane, sum);
            } else if (n == 2) {
                const uint32_t* const x2[2] = {xs[0], xs[1]};
                gateup_rows<CPL, 2>(chunk, at, next, x2, lane, sum);
            } else {
                gateup_rows<CPL, FE_TB>(chunk, at, next, xs, lane, sum);
            }
            if constexpr (APART) {
                const float4 c = apart_products<CPL>(a, s_apart, s_dyn, t0, tok[0] | tok[1] << 8 | tok[2] << 16 | tok[3] << 24,
                                                     e, row, make_float4(sum[0], sum[1], sum[2], sum[3]), lane);
                sum[0] = c.x;
                sum[1] = c.y;
                sum[2] = c.z;
                sum[3] = c.w;
            }
#pragma unroll
            for (int i = 0; i < FE_TB; ++i) {
                if (i >= n) break;
                const int t = t0 + tok[i];
                int j = k;
                if (e != E) j = __ffs(__ballot_sync(0xffffffffu, lane < k && s_idx[t * k + lane] == e)) - 1;
                float g = sum[i];
#pragma unroll
                for (int o = 4; o > 0; o >>= 1) g += __shfl_xor_sync(0xffffffffu, g, o);
                const float u = __shfl_down_sync(0xffffffffu, g, 8);
                if ((lane & 15) == 0) a.h[((int64_t)t * slots + j) * f + row + (lane >> 4)] = g / (1.0f + expf(-g)) * u;
            }
            at = next;
        }
    };
    // two loops: the call takes registers from the one that has it (16 tokens, 256 experts: 78 us, 80 with one).
    // Four outliers in every token make 77 us 95, a single token's 19.6 us 24.2.
    if (!s_apart.any) {
        gate_up(std::false_type());
    } else {
        list_apart<CPL>(s_apart, s_dyn, a.xap + (int64_t)t0 * d, nt);
        gate_up(std::true_type());
    }
    const FewRouting routing{s_idx, s_gate, s_share};
    down_phase<BPQ>(a, d, routing, s_dyn, s_part, s_hblk, &s_ok);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
constexpr size_t FEW_X_BYTES = 180 * 1024;  // inputs of the tokens a CTA keeps for gate/up

struct FewBufs {
    float *logits, *eps, *exact, *h;
    uint32_t *xfix, *bar;
    float* xap;
    size_t bytes;
};
FewBufs few_carve(const pi_moe_layer* L, int64_t T, char* base) {
    PiBump b{base};
    FewBufs o;
    o.bar = b.take<uint32_t>(2);
    o.logits = b.take<float>(T * (L->E + 1));
    o.eps = b.take<float>(T * (L->E + 1));
    o.exact = b.take<float>(T * (L->E + 1));
    o.xfix = b.take<uint32_t>(T * (L->d / 32) * FX_WORDS);
    o.xap = b.take<float>(T * L->d);
    o.h = b.take<float>(T * (L->k + (L->has_shared ? 1 : 0)) * L->f);
    o.bytes = b.off + 256;
    return o;
}

template <int CPL, int NPL, int BPQ>
cudaError_t launch_experts(const FewExpertArgs& a, int sms, cudaStream_t st) {
    const size_t x = (size_t)a.group * (a.d / 32) * FX_WORDS * 4;
    const size_t h = (size_t)(a.k + a.has_shared) * (a.f / 32 * FX_WORDS + 16) * 4, smem = std::max(x, h);
    auto kern = k_few_experts<CPL, NPL, BPQ>;
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

template <int CPL, int NPL>
cudaError_t launch_width(const FewExpertArgs& a, int sms, cudaStream_t st) {
    switch (a.f) {
        case 128: return launch_experts<CPL, NPL, 1>(a, sms, st);
        case 256: return launch_experts<CPL, NPL, 2>(a, sms, st);
        case 512: return launch_experts<CPL, NPL, 4>(a, sms, st);
        default: return launch_experts<CPL, NPL, 8>(a, sms, st);
    }
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
    if (x != out && x < out + T * L->d && out < x + T * L->d)  // a row would be written before another CTA reads it
        return pi_set_error(ctx, PI_ERR_ARG, "moe fused: out may be x, but not overlap it otherwise");
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
        // rows of a CTA: two at least, more where that still gives every SM a CTA and the rows fit
        const int64_t sms = ctx->sm_count > 0 ? ctx->sm_count : 148, groups = (T + FL_GROUP - 1) / FL_GROUP;
        const size_t row = sizeof(float) * (size_t)(d + 128);
        const int fit = (int)(FL_SMEM / row) - FL_GROUP;
        const int R = (int)std::min<int64_t>(fit, std::max<int64_t>(2, ((E + 1) * groups + sms - 1) / sms));
        const size_t smem = row * (FL_GROUP + R);
        pi_smem_attr((const void*)k_few_logits, smem);
        const FewLogitArgs a{x, L->router, L->bias, (int)T, d, E, R, norm ? 1 : 0, B.logits, B.eps, B.xfix, B.bar,
                             B.xap};
        pi_pdl_launch(k_few_logits, dim3((unsigned)((E + R) / R), (unsigned)groups), dim3(FL_T), smem, st, a);
        if (int rc = pi_cuda_check(ctx, cudaGetLastError(), "moe fused logits")) return rc;
    }
    PiProfScope ps(ctx, st, "k_few_experts");
    // as few groups of tokens as fit, of even size, since the CTAs are shared out evenly (n_embd 4096,
    // where 12 fit, 13 tokens of 64 experts: 93 us as 12 + 1, 70 as 7 + 6)
    const int64_t fit = (int64_t)(FEW_X_BYTES / (d / 32 * FX_WORDS * 4)), parts = (T + fit - 1) / fit;
    const int group = (int)((T + parts - 1) / parts);
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
    a.xfix = B.xfix;
    a.xap = B.xap;
    a.logits = B.logits;
    a.eps = B.eps;
    a.exact = B.exact;
    a.router = L->router;
    a.bias = L->bias;
    a.norm = norm ? 1 : 0;
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
        case 1: e = wide ? launch_width<1, 16>(a, sms, st) : launch_width<1, 8>(a, sms, st); break;
        case 2: e = wide ? launch_width<2, 16>(a, sms, st) : launch_width<2, 8>(a, sms, st); break;
        default: e = wide ? launch_width<4, 16>(a, sms, st) : launch_width<4, 8>(a, sms, st); break;
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
