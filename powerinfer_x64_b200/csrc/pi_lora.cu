// A projection over GGUF weights shared by a batch of tokens, beside the low-rank adapters
// of the requests the tokens belong to (no reference counterpart: the reference runs one
// matvec per token, src/quant/mod.rs:939-970, and has no adapters):
//   y_t = W x_t + s_a B_a (A_a x_t),   a = the adapter of token t (none: the first term).
// Q8_0 weights: x is quantised to Q8_0 as in every Q8_0 matvec of the reference
// (:698-736), the 32-element block dots are exact integers, and a block adds
// sumi * (d_w d_x) with one fused multiply-add in f32. Q4_0 weights: f32 x, split into two
// f16 terms at a power-of-two scale per token (22 bits of every value, 40 below the
// token's largest), block dots of the integer nibbles in f32, one fused multiply-add with
// d_w per block. The adapters' products are f32 sums over unquantised x.
//
// Two launches: k_proj_prep (activations in the matrix instructions' fragment order, and
// h_t = s_a A_a x_t), then k_proj_gemm (W's products, B_a h_t added to each output as it
// is stored).
#include "pi_common.cuh"
#include "pi_internal.h"

#include <cuda_bf16.h>

#include <algorithm>
#include <exception>

struct pi_proj {
    pi_ctx* ctx = nullptr;
    int qtype = 0;
    int64_t n_in = 0, n_out = 0;
    int64_t groups = 0;  // groups of four 32-element blocks of a row, the last padded with zeros
    int64_t tiles = 0;   // tiles of 16 rows, an even number, padded with zero rows
    uint8_t* w = nullptr;
};

namespace {

// ---------------------------------------------------------------------------
// Weights in fragment order: [tile of 16 rows][group of 4 blocks], a group being one
// contiguous run that the 32 lanes read with 16-byte loads. Lane 4 g + i holds rows g and
// g + 8 of the tile:
//   Q8_0: 4 x 512 B, per block the lane's {row g: k 4i.., row g+8: k 4i.., row g: k 16+4i..,
//         row g+8: k 16+4i..} (the A registers of m16n8k32)
//   Q4_0: 2 x 512 B, per two blocks the lane's {row g, row g+8} words of k 8i..8i+7, the
//         nibble of k = 8i + 2p (+1) at bits 4p (16 + 4p): one mask then gives a pair of
//         neighbours in the two halves of a register
//   then 128 B of scales: [g][block]{d of row g, d of row g+8} in f16
// ---------------------------------------------------------------------------
template <int QT>
constexpr int group_bytes() { return (QT == PI_QT_Q8_0 ? 2048 : 1024) + 128; }

PI_DEV uint32_t ld_u16x2(const uint8_t* p) {  // GGUF blocks are 2-byte aligned
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
    return q[0] | ((uint32_t)q[1] << 16);
}

// One thread per (tile, group, block, lane); raw holds rows [row0, row0 + rows).
template <int QT>
__global__ __launch_bounds__(128) void k_proj_pack(const uint8_t* __restrict__ raw, int64_t nb, int64_t n_rows,
                                                   int64_t groups, uint8_t* __restrict__ dst) {
    const int b4 = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, i = lane & 3;
    const int64_t tile = blockIdx.x / groups, grp = blockIdx.x % groups, b = grp * 4 + b4;
    constexpr int BB = QT == PI_QT_Q8_0 ? 34 : 18;
    uint8_t* out = dst + (int64_t)blockIdx.x * group_bytes<QT>();
    uint32_t w[2][2] = {{0, 0}, {0, 0}};  // [row g / g + 8][word]
    uint16_t d[2] = {0, 0};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int64_t row = tile * 16 + g + 8 * h;
        if (row >= n_rows || b >= nb) continue;
        const uint8_t* blk = raw + (row * nb + b) * BB;
        d[h] = *reinterpret_cast<const uint16_t*>(blk);
        if (QT == PI_QT_Q8_0) {
            w[h][0] = ld_u16x2(blk + 2 + 4 * i);
            w[h][1] = ld_u16x2(blk + 2 + 16 + 4 * i);
        } else {
            // bytes 4i..4i+3 hold k = 8i..8i+7: byte p is {k = 8i+2p low, k = 8i+2p+1 high}
            const uint32_t v = ld_u16x2(blk + 2 + 4 * i);
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                w[h][0] |= ((v >> (8 * p)) & 15u) << (4 * p);
                w[h][0] |= ((v >> (8 * p + 4)) & 15u) << (16 + 4 * p);
            }
        }
    }
    if (QT == PI_QT_Q8_0) {
        *reinterpret_cast<uint4*>(out + b4 * 512 + lane * 16) = make_uint4(w[0][0], w[1][0], w[0][1], w[1][1]);
    } else {
        *reinterpret_cast<uint2*>(out + (b4 >> 1) * 512 + lane * 16 + (b4 & 1) * 8) = make_uint2(w[0][0], w[1][0]);
    }
    if (i == 0)
        *reinterpret_cast<uint32_t*>(out + group_bytes<QT>() - 128 + g * 16 + b4 * 4) =
            d[0] | ((uint32_t)d[1] << 16);
}

// ---------------------------------------------------------------------------
// Adapters
// ---------------------------------------------------------------------------
struct LoraArgs {
    const void* a;  // [n][R][n_in]
    const void* b;  // [n][n_out][R]
    const int32_t* ranks;
    const float* scales;
    const int32_t* ids;  // [T]
    int dtype, n, R;
};

// Adapter of token t and its rank; -1 where it has none.
PI_DEV int lora_of(const LoraArgs& L, int64_t t, int* rank) {
    const int a = L.ids[t];
    if (a < 0 || a >= L.n) return -1;
    *rank = L.ranks ? min(max(L.ranks[a], 0), L.R) : L.R;
    return a;
}

// eight consecutive adapter weights as f32 (p is 16-byte aligned)
PI_DEV void ld_adapter8(const void* base, int64_t off, int dtype, float* f) {
    if (dtype == PI_QT_F32) {
        const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + off);
        const float4 u = __ldg(p), v = __ldg(p + 1);
        f[0] = u.x; f[1] = u.y; f[2] = u.z; f[3] = u.w;
        f[4] = v.x; f[5] = v.y; f[6] = v.z; f[7] = v.w;
        return;
    }
    const uint4 q = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(base) + off));
    const uint32_t r[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (dtype == PI_QT_F16) {
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&r[i]));
            f[2 * i] = v.x;
            f[2 * i + 1] = v.y;
        } else {
            f[2 * i] = __uint_as_float(r[i] << 16);
            f[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
        }
    }
}

// ---------------------------------------------------------------------------
// k_proj_prep: CTAs 0..T-1 put one token's activations in fragment order (n-tiles of 8
// tokens; lane 4 (t % 8) + i), the CTAs after them one warp per token and four rank rows
// of h. Padded blocks of a row are zero; the columns of tokens behind the last one hold
// whatever the buffer held, and no output reads them (a column of a product depends on
// that column alone).
//   Q8_0: xf [block][n-tile][lane]{k 4i.., k 16+4i..}, xs [block][8 n-tiles] scales
//   Q4_0: xf [block][n-tile][k-step][lane]{hi, hi, lo, lo} (k 8i + 4 step ..), xs [8 n-tiles]
// ---------------------------------------------------------------------------
constexpr int PREP_T = 256;
constexpr int PREP_R = 4;  // rank rows per warp

PI_DEV float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <int QT>
__global__ __launch_bounds__(PREP_T) void k_proj_prep(const float* __restrict__ x, int64_t T, int64_t n_in,
                                                      int64_t groups, int64_t ntt, uint8_t* __restrict__ xf,
                                                      float* __restrict__ xs, const LoraArgs L,
                                                      float* __restrict__ h, uint32_t* err) {
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (blockIdx.x < T) {
        const int64_t t = blockIdx.x, nt = t >> 3;
        const int g = (int)(t & 7);
        const float* xr = x + t * n_in;
        if (L.ids && tid == 0) {
            const int a = L.ids[t];
            if (a >= L.n) atomicOr(err, PI_DEVERR_INDEX);
        }
        if constexpr (QT == PI_QT_Q8_0) {
            for (int64_t c = warp; c < groups; c += PREP_T / 32) {
                const int64_t k = c * 128 + lane * 4;
                float e[4] = {0.f, 0.f, 0.f, 0.f};
                if (k < n_in) {
                    const float4 v = *reinterpret_cast<const float4*>(xr + k);
                    e[0] = v.x; e[1] = v.y; e[2] = v.z; e[3] = v.w;
                }
                float sc;
                const uint32_t q = quad_quant_q8(e, &sc);
                const int64_t blk = c * 4 + (lane >> 3);
                const int j = lane & 7;
                reinterpret_cast<uint32_t*>(xf)[((blk * ntt + nt) * 32 + g * 4 + (j & 3)) * 2 + (j >> 2)] = q;
                if (j == 0) xs[blk * ntt * 8 + t] = sc;
            }
        } else {
            __shared__ float s_m[PREP_T / 32];
            float m = 0.0f;
            for (int64_t k = tid * 4; k < n_in; k += PREP_T * 4) {
                const float4 v = *reinterpret_cast<const float4*>(xr + k);
                m = max_nan(m, max_nan(max_nan(fabsf(v.x), fabsf(v.y)), max_nan(fabsf(v.z), fabsf(v.w))));
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (lane == 0) s_m[warp] = m;
            __syncthreads();
            for (int i = 0; i < PREP_T / 32; ++i) m = max_nan(m, s_m[i]);
            // 2^e with max |x| 2^e in [2^13, 2^14): the products stay far from f16's and f32's
            // limits; a NaN or infinity makes the whole token NaN
            const int ex = m > 0.0f ? min(13 - ilogbf(m), 120) : 0;
            const bool fin = m < INFINITY;
            const float s = fin ? ldexpf(1.0f, ex) : __int_as_float(0x7fffffff);
            if (tid == 0) xs[t] = fin ? ldexpf(1.0f, -ex) : __int_as_float(0x7fffffff);
            for (int64_t j = tid; j < groups * 16; j += PREP_T) {
                float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (j * 8 < n_in) {
                    const float4 u = *reinterpret_cast<const float4*>(xr + j * 8);
                    const float4 w = *reinterpret_cast<const float4*>(xr + j * 8 + 4);
                    v[0] = u.x * s; v[1] = u.y * s; v[2] = u.z * s; v[3] = u.w * s;
                    v[4] = w.x * s; v[5] = w.y * s; v[6] = w.z * s; v[7] = w.w * s;
                }
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const __half2 a = __floats2half2_rn(v[2 * p], v[2 * p + 1]);
                    const float2 b = __half22float2(a);
                    const __half2 c = __floats2half2_rn(v[2 * p] - b.x, v[2 * p + 1] - b.y);
                    hi[p] = *reinterpret_cast<const uint32_t*>(&a);
                    lo[p] = *reinterpret_cast<const uint32_t*>(&c);
                }
                uint4* o = reinterpret_cast<uint4*>(xf) + ((j >> 2) * ntt + nt) * 64 + g * 4 + (j & 3);
                o[0] = make_uint4(hi[0], hi[1], lo[0], lo[1]);
                o[32] = make_uint4(hi[2], hi[3], lo[2], lo[3]);
            }
        }
        return;
    }
    // h[t][r] = scale * (A[a][r] . x[t])
    const int per = L.R / PREP_R;
    const int64_t w = (blockIdx.x - T) * (PREP_T / 32) + warp, t = w / per;
    const int r0 = (int)(w % per) * PREP_R;
    if (t >= T) return;
    int rank;
    const int a = lora_of(L, t, &rank);
    if (a < 0 || r0 >= rank) return;
    float acc[PREP_R] = {};
    const float* xr = x + t * n_in;
    const int64_t base = ((int64_t)a * L.R + r0) * n_in;
#pragma unroll 2
    for (int64_t k = lane * 8; k < n_in; k += 256) {
        const float4 u = *reinterpret_cast<const float4*>(xr + k);
        const float4 v = *reinterpret_cast<const float4*>(xr + k + 4);
#pragma unroll
        for (int r = 0; r < PREP_R; ++r) {
            float f[8];
            ld_adapter8(L.a, base + r * n_in + k, L.dtype, f);
            acc[r] = fmaf(f[0], u.x, acc[r]);
            acc[r] = fmaf(f[1], u.y, acc[r]);
            acc[r] = fmaf(f[2], u.z, acc[r]);
            acc[r] = fmaf(f[3], u.w, acc[r]);
            acc[r] = fmaf(f[4], v.x, acc[r]);
            acc[r] = fmaf(f[5], v.y, acc[r]);
            acc[r] = fmaf(f[6], v.z, acc[r]);
            acc[r] = fmaf(f[7], v.w, acc[r]);
        }
    }
    const float sc = L.scales ? L.scales[a] : 1.0f;
#pragma unroll
    for (int r = 0; r < PREP_R; ++r) {
        const float s = warp_sum(acc[r]);
        if (lane == 0) h[t * L.R + r0 + r] = s * sc;
    }
}

// ---------------------------------------------------------------------------
// k_proj_gemm
// ---------------------------------------------------------------------------
struct ProjArgs {
    const uint8_t* w;
    const uint8_t* xf;
    const float* xs;
    const float* h;
    float* y;
    LoraArgs L;
    int64_t T, n_out, groups, tiles, ntt;
    int ks;  // warps that share a tile's blocks
};

PI_DEV uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
PI_DEV float2 unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
PI_DEV uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
PI_DEV uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
PI_DEV uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// 1.5 * 2^23 as bits: an integer sum below 2^22 added to these bits is the float
// 1.5 * 2^23 + sum, so accumulating on it replaces the conversion by one subtraction.
constexpr int FLOAT_BIAS_BITS = 0x4B400000;
constexpr float FLOAT_BIAS = 12582912.0f;

PI_DEV void mma_s8(int (&c)[4], const uint4& a, const uint2& b) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(FLOAT_BIAS_BITS));
}
PI_DEV void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// nibbles p and p + 4 of a word as f16 values n - 8 (1024 + n is exact; so is 1024 + n - 1032)
PI_DEV uint32_t nib_pair(uint32_t w, int p) {
    uint32_t v;
    asm("lop3.b32 %0, %1, 0x000F000F, 0x64006400, 0xEA;" : "=r"(v) : "r"(w >> (4 * p)));
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v), __half2half2(__ushort_as_half(0x6408)));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// A lane's words of one group of MT tiles.
template <int QT, int MT>
struct GroupRegs {
    static constexpr int NQ = QT == PI_QT_Q8_0 ? 4 : 2;
    int4 q[MT][NQ];
    int4 d[MT];
    PI_DEV void load(const uint8_t* p, int64_t tile_stride, int lane) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
            for (int i = 0; i < NQ; ++i) q[m][i] = ld_stream(p + m * tile_stride + i * 512 + lane * 16);
            d[m] = ld_stream(p + m * tile_stride + NQ * 512 + (lane >> 2) * 16);
        }
    }
};
PI_DEV int word(const int4& v, int i) { return i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w)); }

// CTA = 8 warps = 8 / ks sets of MT tiles, each set's blocks split over ks warps; NT n-tiles
// of 8 tokens (blockIdx.y: which). The weights stream from memory once per 8 NT tokens,
// the next group's 16-byte loads in flight while the current one is multiplied; the
// activations' fragments are read through L1, which the weights bypass.
template <int QT, int MT, int NT>
__global__ __launch_bounds__(256) void k_proj_gemm(const ProjArgs p) {
    extern __shared__ __align__(16) float s_red[];  // [warp][MT * NT][4][32] when ks > 1
    __shared__ int s_id[8 * NT], s_rank[8 * NT];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, i4 = lane & 3;
    const int ks = p.ks, part = warp % ks;
    const int64_t set = (int64_t)blockIdx.x * (8 / ks) + warp / ks, tile0 = set * MT;
    const int64_t nt0 = (int64_t)blockIdx.y * NT;
    const int nnt = (int)min((int64_t)NT, p.ntt - nt0);  // n-tiles of this CTA
    const int64_t tile_stride = p.groups * group_bytes<QT>();
    const int64_t gb = p.groups * part / ks, ge = p.groups * (part + 1) / ks;
    const bool live = tile0 < p.tiles;
    const uint8_t* wp = p.w + tile0 * tile_stride + gb * group_bytes<QT>();
    GroupRegs<QT, MT> cur, nxt;
    if (live && gb < ge) cur.load(wp, tile_stride, lane);  // constant weights: before the wait
    pdl_wait();
    pdl_trigger();
    for (int j = tid; j < 8 * NT; j += 256) {
        const int64_t t = nt0 * 8 + j;
        int rank = 0;
        s_id[j] = (p.L.ids && t < p.T) ? lora_of(p.L, t, &rank) : -1;
        s_rank[j] = rank;
    }
    uint64_t acc[MT][NT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n][0] = acc[m][n][1] = 0;
    if (live) {
        for (int64_t gr = gb; gr < ge; ++gr) {
            wp += group_bytes<QT>();
            if (gr + 1 < ge) nxt.load(wp, tile_stride, lane);
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                uint64_t dg[MT][2];  // {d, d} of rows g and g + 8
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const int w = word(cur.d[m], b);
                    const float2 d = __half22float2(*reinterpret_cast<const __half2*>(&w));
                    dg[m][0] = pack2(d.x, d.x);
                    dg[m][1] = pack2(d.y, d.y);
                }
                const int64_t blk = gr * 4 + b;
                if constexpr (QT == PI_QT_Q8_0) {
                    const uint2* xb = reinterpret_cast<const uint2*>(p.xf) + (blk * p.ntt + nt0) * 32 + lane;
                    const uint64_t* db = reinterpret_cast<const uint64_t*>(p.xs + (blk * p.ntt + nt0) * 8 + 2 * i4);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        if (n >= nnt) break;
                        const uint2 xv = xb[n * 32];
                        const uint64_t dx = db[n * 4];
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            int c[4];
                            mma_s8(c, *reinterpret_cast<const uint4*>(&cur.q[m][b]), xv);
                            const uint64_t bias = pack2(-FLOAT_BIAS, -FLOAT_BIAS);
                            const uint64_t f0 = add2(pack2(__int_as_float(c[0]), __int_as_float(c[1])), bias);
                            const uint64_t f1 = add2(pack2(__int_as_float(c[2]), __int_as_float(c[3])), bias);
                            acc[m][n][0] = fma2(f0, mul2(dg[m][0], dx), acc[m][n][0]);
                            acc[m][n][1] = fma2(f1, mul2(dg[m][1], dx), acc[m][n][1]);
                        }
                    }
                } else {
                    uint32_t a[MT][2][4];
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        const uint32_t w0 = word(cur.q[m][b >> 1], 2 * (b & 1));
                        const uint32_t w1 = word(cur.q[m][b >> 1], 2 * (b & 1) + 1);
#pragma unroll
                        for (int s = 0; s < 2; ++s) {
                            a[m][s][0] = nib_pair(w0, 2 * s);
                            a[m][s][1] = nib_pair(w1, 2 * s);
                            a[m][s][2] = nib_pair(w0, 2 * s + 1);
                            a[m][s][3] = nib_pair(w1, 2 * s + 1);
                        }
                    }
                    const uint4* xb = reinterpret_cast<const uint4*>(p.xf) + (blk * p.ntt + nt0) * 64 + lane;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        if (n >= nnt) break;
                        const uint4 x0 = xb[n * 64], x1 = xb[n * 64 + 32];
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            float c[4] = {0.f, 0.f, 0.f, 0.f};
                            mma_f16(c, a[m][0], x0.z, x0.w);
                            mma_f16(c, a[m][1], x1.z, x1.w);
                            mma_f16(c, a[m][0], x0.x, x0.y);
                            mma_f16(c, a[m][1], x1.x, x1.y);
                            acc[m][n][0] = fma2(dg[m][0], pack2(c[0], c[1]), acc[m][n][0]);
                            acc[m][n][1] = fma2(dg[m][1], pack2(c[2], c[3]), acc[m][n][1]);
                        }
                    }
                }
            }
            cur = nxt;
        }
    }
    if (ks > 1) {
        float* mine = s_red + (size_t)warp * (MT * NT * 128) + lane;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (n >= nnt) break;
                const float2 u = unpack2(acc[m][n][0]), v = unpack2(acc[m][n][1]);
                float* o = mine + (m * NT + n) * 128;
                o[0] = u.x;
                o[32] = u.y;
                o[64] = v.x;
                o[96] = v.y;
            }
    }
    __syncthreads();
    if (!live) return;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (n >= nnt) break;
            if (ks > 1 && n % ks != part) continue;
            float c[2][2];  // [row g / g + 8][token 2 i4, 2 i4 + 1]
            if (ks > 1) {
                const float* from = s_red + (size_t)(warp - part) * (MT * NT * 128) + (m * NT + n) * 128 + lane;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float s = 0.0f;
                    for (int q = 0; q < ks; ++q) s += from[(size_t)q * (MT * NT * 128) + j * 32];
                    c[j >> 1][j & 1] = s;
                }
            } else {
                const float2 u = unpack2(acc[m][n][0]), v = unpack2(acc[m][n][1]);
                c[0][0] = u.x;
                c[0][1] = u.y;
                c[1][0] = v.x;
                c[1][1] = v.y;
            }
            const int64_t row = (tile0 + m) * 16 + g;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int j = n * 8 + 2 * i4 + e;
                const int64_t t = nt0 * 8 + j;
                if (t >= p.T) continue;
                if (QT == PI_QT_Q4_0) {
                    const float s = p.xs[t];
                    c[0][e] *= s;
                    c[1][e] *= s;
                }
                const int a = s_id[j], rank = s_rank[j];
                if (a >= 0) {
                    const float* h = p.h + t * p.L.R;
                    for (int r = 0; r < rank; r += 8) {
                        float hv[8];
#pragma unroll
                        for (int q = 0; q < 8; ++q) hv[q] = r + q < rank ? h[r + q] : 0.0f;
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            if (row + 8 * k >= p.n_out) continue;
                            float f[8];
                            ld_adapter8(p.L.b, ((int64_t)a * p.n_out + row + 8 * k) * p.L.R + r, p.L.dtype, f);
#pragma unroll
                            for (int q = 0; q < 8; ++q)
                                if (r + q < rank) c[k][e] = fmaf(f[q], hv[q], c[k][e]);
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    if (row + 8 * k < p.n_out) p.y[t * p.n_out + row + 8 * k] = c[k][e];
            }
        }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
int64_t proj_raw_bytes(int qtype, int64_t n) { return n / 32 * (qtype == PI_QT_Q8_0 ? 34 : 18); }

struct ProjBufs {
    uint8_t* xf;
    float *xs, *h;
    size_t bytes;
};
ProjBufs proj_carve(const pi_proj* P, int64_t T, int64_t R, char* base) {
    PiBump b{base};
    ProjBufs o;
    const int64_t ntt = (T + 7) / 8, blocks = P->groups * 4;
    o.xf = b.take<uint8_t>((size_t)(blocks * ntt) * (P->qtype == PI_QT_Q8_0 ? 256 : 1024));
    o.xs = b.take<float>((size_t)(ntt * 8) * (P->qtype == PI_QT_Q8_0 ? blocks : 1));
    o.h = b.take<float>((size_t)(T * R));
    o.bytes = b.off + 256;
    return o;
}

template <int QT>
int proj_pack(pi_ctx* ctx, pi_proj* P, const uint8_t* raw, int src_on_host) {
    const int64_t nb = P->n_in / 32, row_bytes = proj_raw_bytes(QT, P->n_in), stride = P->groups * group_bytes<QT>();
    // a host source comes over in runs of whole tiles, 64 MB at most
    const int64_t per = src_on_host ? std::max<int64_t>(1, (64 << 20) / (16 * row_bytes)) : P->tiles;
    uint8_t* stage = nullptr;
    if (src_on_host &&
        pi_cuda_check(ctx, cudaMalloc(&stage, (size_t)(std::min(per, P->tiles) * 16 * row_bytes)), "cudaMalloc(stage)"))
        return PI_ERR_OOM;
    int rc = PI_OK;
    for (int64_t t = 0; t < P->tiles && !rc; t += per) {
        const int64_t nt = std::min(per, P->tiles - t), rows = std::max<int64_t>(0, std::min(P->n_out - t * 16, nt * 16));
        const uint8_t* src = raw + t * 16 * row_bytes;
        if (src_on_host && rows) {
            if (pi_cuda_check(ctx, cudaMemcpy(stage, src, (size_t)(rows * row_bytes), cudaMemcpyHostToDevice), "upload"))
                rc = PI_ERR_CUDA;
            src = stage;
        }
        if (rc) break;
        k_proj_pack<QT><<<(unsigned)(nt * P->groups), 128>>>(src, nb, rows, P->groups, P->w + t * stride);
        if (pi_cuda_check(ctx, cudaDeviceSynchronize(), "projection pack")) rc = PI_ERR_CUDA;
    }
    if (stage) cudaFree(stage);
    return rc;
}

int proj_create(pi_ctx* ctx, const void* raw, uint64_t raw_len, int32_t qtype, int64_t n_in, int64_t n_out,
                int32_t src_on_host, pi_proj** out) {
    if (qtype != PI_QT_Q8_0 && qtype != PI_QT_Q4_0)
        return pi_set_error(ctx, PI_ERR_ARG, "projection: weights must be Q8_0 or Q4_0");
    if (n_in < 32 || n_in % 32 || n_in > (1 << 20) || n_out < 1 || n_out > (1 << 24))
        return pi_set_error(ctx, PI_ERR_ARG, "projection: need n_in a multiple of 32 up to 2^20 and 1 <= n_out <= 2^24");
    if (!raw || !out) return pi_set_error(ctx, PI_ERR_ARG, "projection: null pointer");
    if (!src_on_host && ((uintptr_t)raw & 1))
        return pi_set_error(ctx, PI_ERR_ARG, "projection: GGUF blocks on the device must be 2-byte aligned");
    if (raw_len < (uint64_t)proj_raw_bytes(qtype, n_in) * (uint64_t)n_out)
        return pi_set_error(ctx, PI_ERR_SHORT, "projection: fewer bytes than n_out rows of n_in values");
    PiDeviceGuard dev(ctx->device);
    pi_proj* P = new pi_proj();
    P->ctx = ctx;
    P->qtype = qtype;
    P->n_in = n_in;
    P->n_out = n_out;
    P->groups = (n_in / 32 + 3) / 4;
    P->tiles = ((n_out + 15) / 16 + 1) & ~(int64_t)1;
    const int64_t gbytes = qtype == PI_QT_Q8_0 ? group_bytes<PI_QT_Q8_0>() : group_bytes<PI_QT_Q4_0>();
    if (P->tiles * P->groups > INT32_MAX) {
        delete P;
        return pi_set_error(ctx, PI_ERR_ARG, "projection: too large");
    }
    int rc = PI_OK;
    if (pi_cuda_check(ctx, cudaMalloc((void**)&P->w, (size_t)(P->tiles * P->groups * gbytes)), "cudaMalloc(projection)"))
        rc = PI_ERR_OOM;
    if (!rc)
        rc = qtype == PI_QT_Q8_0 ? proj_pack<PI_QT_Q8_0>(ctx, P, (const uint8_t*)raw, src_on_host)
                                 : proj_pack<PI_QT_Q4_0>(ctx, P, (const uint8_t*)raw, src_on_host);
    if (rc) {
        pi_proj_destroy(P);
        return rc;
    }
    *out = P;
    return PI_OK;
}

template <int QT, int MT, int NT>
void launch_gemm(const ProjArgs& a, cudaStream_t st) {
    const size_t smem = a.ks > 1 ? sizeof(float) * 8 * MT * NT * 128 : 0;
    pi_smem_attr((const void*)k_proj_gemm<QT, MT, NT>, smem);
    const int64_t per = (int64_t)MT * (8 / a.ks);
    pi_pdl_launch(k_proj_gemm<QT, MT, NT>,
                  dim3((unsigned)((a.tiles + per - 1) / per), (unsigned)((a.ntt + NT - 1) / NT)), dim3(256), smem, st, a);
}

template <int QT>
void dispatch_gemm(ProjArgs a, int64_t sms, cudaStream_t st) {
    // Two tiles per warp halve the activation reads from L1, which bound batches of more
    // than 16 tokens, where enough tiles are left to fill the SMs with 8 warps each
    if (a.ntt > 2 && a.tiles / 2 >= 8 * sms) {
        a.ks = 1;
        if (a.ntt <= 4) launch_gemm<QT, 2, 4>(a, st);
        else launch_gemm<QT, 2, 8>(a, st);
        return;
    }
    // Few rows: a tile's blocks are split over up to eight warps, until 16 warps per SM
    // have work
    a.ks = 1;
    while (a.ks < 8 && a.tiles * a.ks < 16 * sms && a.groups >= 2 * a.ks) a.ks *= 2;
    if (a.ntt <= 1) launch_gemm<QT, 1, 1>(a, st);
    else if (a.ntt <= 2) launch_gemm<QT, 1, 2>(a, st);
    else if (a.ntt <= 4) launch_gemm<QT, 1, 4>(a, st);
    else launch_gemm<QT, 1, 8>(a, st);
}

int check_bank(pi_ctx* ctx, const pi_lora_bank* bank, const int32_t* ids) {
    if (!bank) return ids ? pi_set_error(ctx, PI_ERR_ARG, "projection: adapter ids without a bank") : PI_OK;
    if (bank->dtype != PI_QT_F32 && bank->dtype != PI_QT_F16 && bank->dtype != PI_QT_BF16)
        return pi_set_error(ctx, PI_ERR_ARG, "adapters: F32, F16 or BF16");
    if (bank->n_adapters < 1 || bank->max_rank < 8 || bank->max_rank > 1024 || bank->max_rank % 8)
        return pi_set_error(ctx, PI_ERR_ARG, "adapters: need one at least, max_rank a multiple of 8 from 8 to 1024");
    if (!bank->a || !bank->b || !ids) return pi_set_error(ctx, PI_ERR_ARG, "adapters: null pointer");
    if (((uintptr_t)bank->a | (uintptr_t)bank->b) & 15)
        return pi_set_error(ctx, PI_ERR_ARG, "adapters: a and b must be 16-byte aligned");
    return PI_OK;
}

int proj_forward(pi_ctx* ctx, const pi_proj* P, const float* x, int64_t T, const pi_lora_bank* bank,
                 const int32_t* ids, float* y, void* workspace, uint64_t workspace_bytes, cudaStream_t st) {
    if (P->ctx->device != ctx->device) return pi_set_error(ctx, PI_ERR_ARG, "projection: made on another device");
    if (T < 0 || T > (1 << 20)) return pi_set_error(ctx, PI_ERR_ARG, "projection: need 0 <= T <= 2^20");
    if (int rc = check_bank(ctx, bank, ids)) return rc;
    if (T == 0) return PI_OK;
    if (!x || !y) return pi_set_error(ctx, PI_ERR_ARG, "projection: null pointer");
    if (((uintptr_t)x & 15) || ((uintptr_t)y & 3) || ((uintptr_t)workspace & 255))
        return pi_set_error(ctx, PI_ERR_ARG, "projection: x must be 16-byte, y 4-byte and the workspace 256-byte aligned");
    const int64_t R = bank ? bank->max_rank : 0;
    const size_t need = proj_carve(P, T, R, nullptr).bytes;
    PiDeviceGuard dev(ctx->device);
    char* scr = (char*)workspace;
    if (workspace && workspace_bytes < need) return pi_set_error(ctx, PI_ERR_SHORT, "projection: workspace too small");
    if (!workspace)
        if (int rc = pi_scratch(ctx, st, need, &scr)) return rc;
    const ProjBufs B = proj_carve(P, T, R, scr);
    LoraArgs L = {};
    if (bank) L = LoraArgs{bank->a, bank->b, bank->ranks, bank->scales, ids, bank->dtype, bank->n_adapters, (int)R};
    const bool q8 = P->qtype == PI_QT_Q8_0;
    const int64_t ntt = (T + 7) / 8;
    {
        PiProfScope ps(ctx, st, "k_proj_prep");
        const int64_t warps = T * (R / PREP_R), grid = T + (warps + PREP_T / 32 - 1) / (PREP_T / 32);
        if (q8)
            pi_pdl_launch(k_proj_prep<PI_QT_Q8_0>, dim3((unsigned)grid), dim3(PREP_T), 0, st, x, T, P->n_in, P->groups,
                          ntt, B.xf, B.xs, L, B.h, ctx->dev_err);
        else
            pi_pdl_launch(k_proj_prep<PI_QT_Q4_0>, dim3((unsigned)grid), dim3(PREP_T), 0, st, x, T, P->n_in, P->groups,
                          ntt, B.xf, B.xs, L, B.h, ctx->dev_err);
    }
    {
        PiProfScope ps(ctx, st, "k_proj_gemm");
        const ProjArgs a{P->w, B.xf, B.xs, B.h, y, L, T, P->n_out, P->groups, P->tiles, ntt, 1};
        const int64_t sms = ctx->sm_count > 0 ? ctx->sm_count : 148;
        if (q8) dispatch_gemm<PI_QT_Q8_0>(a, sms, st);
        else dispatch_gemm<PI_QT_Q4_0>(a, sms, st);
    }
    return pi_cuda_check(ctx, cudaGetLastError(), "projection") ? PI_ERR_CUDA : PI_OK;
}

}  // namespace

extern "C" int pi_proj_create(pi_ctx* ctx, const void* raw, uint64_t raw_len, int32_t qtype, int64_t n_in,
                              int64_t n_out, int32_t src_on_host, pi_proj** out) {
    if (!ctx) return PI_ERR_ARG;
    if (out) *out = nullptr;
    try {
        return proj_create(ctx, raw, raw_len, qtype, n_in, n_out, src_on_host, out);
    } catch (const std::exception&) {  // an allocation of the host failed
        return PI_ERR_OOM;
    }
}

extern "C" void pi_proj_destroy(pi_proj* P) {
    if (!P) return;
    PiDeviceGuard dev(P->ctx->device);
    if (P->w) cudaFree(P->w);
    delete P;
}

extern "C" uint64_t pi_proj_workspace(const pi_proj* P, int64_t T, const pi_lora_bank* bank) {
    return P && T > 0 ? proj_carve(P, T, bank ? bank->max_rank : 0, nullptr).bytes : 0;
}

extern "C" int pi_proj_forward(pi_ctx* ctx, const pi_proj* P, const float* x, int64_t T, const pi_lora_bank* bank,
                               const int32_t* adapter_ids, float* y, void* workspace, uint64_t workspace_bytes,
                               void* stream) {
    if (!ctx || !P) return PI_ERR_ARG;
    try {
        return proj_forward(ctx, P, x, T, bank, adapter_ids, y, workspace, workspace_bytes, (cudaStream_t)stream);
    } catch (const std::exception&) {
        return PI_ERR_OOM;
    }
}
