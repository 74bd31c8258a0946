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
// Up to three launches: k_proj_prep (activations in the matrix instructions' fragment order,
// and h_t = s_a A_a x_t), k_proj_gemm (W's products), k_proj_adapters (B_a h_t added).
#include "pi_common.cuh"
#include "pi_internal.h"

#include <cooperative_groups.h>

#include <algorithm>
#include <exception>
#include <map>

namespace cg = cooperative_groups;

struct pi_proj {
    pi_ctx* ctx = nullptr;
    int qtype = 0;
    int64_t n_in = 0, n_out = 0;
    int64_t units = 0;   // pairs of 32-element blocks of a row, the last padded with zeros
    int64_t tiles = 0;   // tiles of 16 rows, the last padded with zero rows
    uint8_t* w = nullptr;
    // how k_proj_gemm is launched for a number of n-tiles, found at its first use
    struct Plan {
        int ks, cu, nchunk, sums;
        size_t smem;
    };
    mutable std::mutex mu;
    mutable std::map<int64_t, Plan> plans;
};

namespace {

// ---------------------------------------------------------------------------
// Weights in fragment order: [tile of 16 rows][unit of 2 blocks], a unit being one contiguous
// run that the 32 lanes read with 16-byte loads. Lane 4 g + i holds rows g and g + 8 of the
// tile:
//   Q8_0: 2 x 512 B, per block the lane's {row g: k 4i.., row g+8: k 4i.., row g: k 16+4i..,
//         row g+8: k 16+4i..} (the A registers of m16n8k32)
//   Q4_0: 512 B, per block the lane's {row g, row g+8} words of k 8i..8i+7, the nibble of
//         k = 8i + 2p (+1) at bits 4p (16 + 4p): one mask then gives a pair of neighbours
//         in the two halves of a register
//   then 64 B of scales: [g][block]{d of row g, d of row g+8} in f16
// ---------------------------------------------------------------------------
template <int QT>
constexpr int unit_bytes() { return (QT == PI_QT_Q8_0 ? 1024 : 512) + 64; }

PI_DEV uint32_t ld_u16x2(const uint8_t* p) {  // GGUF blocks are 2-byte aligned
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
    return q[0] | ((uint32_t)q[1] << 16);
}

// One thread per (tile, unit, block, lane); raw holds n_rows rows.
template <int QT>
__global__ __launch_bounds__(64) void k_proj_pack(const uint8_t* __restrict__ raw, int64_t nb, int64_t n_rows,
                                                  int64_t units, uint8_t* __restrict__ dst) {
    const int b2 = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, i = lane & 3;
    const int64_t tile = blockIdx.x / units, unit = blockIdx.x % units, b = unit * 2 + b2;
    constexpr int BB = QT == PI_QT_Q8_0 ? 34 : 18;
    uint8_t* out = dst + (int64_t)blockIdx.x * unit_bytes<QT>();
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
        *reinterpret_cast<uint4*>(out + b2 * 512 + lane * 16) = make_uint4(w[0][0], w[1][0], w[0][1], w[1][1]);
    } else {
        *reinterpret_cast<uint2*>(out + lane * 16 + b2 * 8) = make_uint2(w[0][0], w[1][0]);
    }
    if (i == 0)
        *reinterpret_cast<uint32_t*>(out + unit_bytes<QT>() - 64 + g * 8 + b2 * 4) = d[0] | ((uint32_t)d[1] << 16);
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
// Activations in fragment order: [chunk of NT n-tiles of 8 tokens][unit of 2 blocks][n-tile],
// so that a run of units of one chunk is one contiguous piece. Lane 4 g + i holds token g of
// the n-tile:
//   Q8_0: 512 B, the lane's {k 4i.., k 16+4i..} of either block, then 64 B of scales, i's
//         {tokens 2i, 2i+1} of either block (f32: as f16 the conversions cost more, 150 us
//         against 137 at n_out 151936 and 64 tokens, than the reads saved)
//   Q4_0: per block and k-step (k 8i + 4 step ..) 512 B, the lane's {hi, hi, lo, lo}
// ---------------------------------------------------------------------------
template <int QT>
constexpr int xunit_bytes() { return QT == PI_QT_Q8_0 ? 512 + 64 : 4 * 512; }

PI_DEV uint32_t to_tf32(float v) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
    return r;
}

// ---------------------------------------------------------------------------
// k_proj_prep: CTAs 0..T-1 put one token's activations in fragment order; the CTAs after
// them compute h, S = 2, 4, 8 or 16 warps per token and four rank rows (a row's parts in turn, 256
// values of each at a time: few tokens take many warps, whose loads are then one or two round
// trips to memory). Padded blocks of a row are zero; the columns of tokens behind the last
// one hold whatever the buffer held, and no output reads them (a column of a product depends
// on it alone).
// Q4_0 activations are scaled by a power of two per token, its reciprocal in xs [T].
// ---------------------------------------------------------------------------
constexpr int PREP_T = 512;
constexpr int PREP_R = 4;   // rank rows of a unit

template <int QT>
__global__ __launch_bounds__(PREP_T) void k_proj_prep(const float* __restrict__ x, int64_t T, int64_t n_in,
                                                      int64_t units, int NT, uint8_t* __restrict__ xf,
                                                      float* __restrict__ xs, const LoraArgs L,
                                                      float* __restrict__ h, int S, uint32_t* err) {
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (blockIdx.x < T) {
        const int64_t t = blockIdx.x, chunk = t / (8 * NT), c0 = chunk * (8 * NT);
        const int col = (int)(t - c0);
        const int g = col & 7;
        const float* xr = x + t * n_in;
        uint8_t* xo = xf + (chunk * units * NT + (col >> 3)) * xunit_bytes<QT>();
        const int64_t ustride = (int64_t)NT * xunit_bytes<QT>();
        if (L.ids && tid == 0) {
            const int a = L.ids[t];
            if (a >= L.n) atomicOr(err, PI_DEVERR_INDEX);
        }
        if constexpr (QT == PI_QT_Q8_0) {
            for (int64_t c = warp; 2 * c < units; c += PREP_T / 32) {  // four blocks
                const int64_t k = c * 128 + lane * 4, u = 2 * c + (lane >> 4);
                float e[4] = {0.f, 0.f, 0.f, 0.f};
                if (k < n_in) {
                    const float4 v = *reinterpret_cast<const float4*>(xr + k);
                    e[0] = v.x; e[1] = v.y; e[2] = v.z; e[3] = v.w;
                }
                float sc;
                const uint32_t q = quad_quant_q8(e, &sc);
                if (u >= units) continue;
                const int b = (lane >> 3) & 1, j = lane & 7;  // eighth j of the unit's block b
                uint8_t* o = xo + u * ustride;
                *reinterpret_cast<uint32_t*>(o + (g * 4 + (j & 3)) * 16 + b * 8 + (j >> 2) * 4) = q;
                if (j == 0) *reinterpret_cast<float*>(o + 512 + (g >> 1) * 16 + b * 8 + (g & 1) * 4) = sc;
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
            for (int64_t j = tid; j < units * 8; j += PREP_T) {  // eight values: lane i = j % 4 of block j / 4
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
                uint8_t* o = xo + (j >> 3) * ustride + ((j >> 2) & 1) * 1024 + (g * 4 + (j & 3)) * 16;
                *reinterpret_cast<uint4*>(o) = make_uint4(hi[0], hi[1], lo[0], lo[1]);
                *reinterpret_cast<uint4*>(o + 512) = make_uint4(hi[2], hi[3], lo[2], lo[3]);
            }
        }
        return;
    }
    // h[t][r] = scale * (A[a][r] . x[t]), zero from the rank on, as two tf32 terms: per unit
    // of four rank rows the four large terms, then the four small ones
    __shared__ float s_h[PREP_T / 32][PREP_R];
    const int per = L.R / PREP_R, part = warp % S;
    const int64_t unit = (blockIdx.x - T) * (PREP_T / 32 / S) + warp / S, t = unit / per;
    const int r0 = (int)(unit % per) * PREP_R;
    int rank = 0, a = -1;
    if (t < T) a = lora_of(L, t, &rank);
    const bool live = a >= 0 && r0 < rank;
    if (live) {
        float acc[PREP_R] = {};
        const float* xr = x + t * n_in;
        const int64_t base = ((int64_t)a * L.R + r0) * n_in;
#pragma unroll 4
        for (int64_t k = part * 256 + lane * 8; k < n_in; k += 256 * S) {
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
#pragma unroll
        for (int r = 0; r < PREP_R; ++r) {
            const float s = warp_sum(acc[r]);
            if (lane == 0) s_h[warp][r] = s;
        }
    }
    __syncthreads();
    if (live && part == 0 && lane < PREP_R) {
        float s = 0.0f;
        for (int q = 0; q < S; ++q) s += s_h[warp + q][lane];
        s = r0 + lane < rank ? s * (L.scales ? L.scales[a] : 1.0f) : 0.0f;
        const uint32_t big = to_tf32(s);
        float* o = h + (t * L.R + r0) * 2 + lane;
        o[0] = __uint_as_float(big);
        o[PREP_R] = __uint_as_float(to_tf32(s - __uint_as_float(big)));
    }
}

// ---------------------------------------------------------------------------
// k_proj_gemm
// ---------------------------------------------------------------------------
struct ProjArgs {
    const uint8_t* w;
    const uint8_t* xf;
    const float* xs;
    float* y;
    int64_t T, n_out, units, tiles;
    int ks;      // CTAs that share the blocks of their rows
    int cu;      // units of a part that are staged together
    int nchunk;  // such pieces of a part
    int sums;    // where the parts' sums lie in shared memory
};

PI_DEV void mma_s8(int (&c)[4], const uint4& a, const uint2& b) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(0));
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

// A lane's words of one unit of a tile.
template <int QT>
struct UnitRegs {
    static constexpr int NQ = QT == PI_QT_Q8_0 ? 2 : 1;
    int4 q[NQ];
    int2 d;
    PI_DEV void load(const uint8_t* p, int lane) {
#pragma unroll
        for (int i = 0; i < NQ; ++i) q[i] = ld_stream(p + i * 512 + lane * 16);
        asm volatile("ld.global.nc.L1::no_allocate.v2.s32 {%0,%1}, [%2];"
                     : "=r"(d.x), "=r"(d.y)
                     : "l"(p + NQ * 512 + (lane >> 2) * 8));
    }
};
PI_DEV int word(const int4& v, int i) { return i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w)); }

PI_DEV void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

PI_DEV void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

constexpr int GEMM_T = 256;
constexpr int GEMM_W = GEMM_T / 32;
constexpr size_t GEMM_SMEM = 200 * 1024;
constexpr int RING = 4;  // units a warp holds or has in flight (4 KB of Q8_0 weights)

// CTA = 8 warps of 16 rows each; blockIdx.x = the CTA's part of the blocks (the ks CTAs of a
// cluster share their rows) + ks * the set of 128 rows; blockIdx.y: the chunk of NT
// n-tiles. The weights stream from memory once per chunk straight into a ring of D units in
// registers; the activations' fragments come through a stage in shared memory that the
// CTA's warps share, double-buffered where a part does not fit. Splitting over CTAs rather
// than over a CTA's warps keeps 128 rows to every staged fragment (n_out 12288, T 16, Q4_0:
// 54 us with the blocks split over the warps, 36 over a cluster).
template <int QT, int NT>
__global__ __launch_bounds__(GEMM_T, 2) void k_proj_gemm(const ProjArgs p) {
    constexpr int XU = xunit_bytes<QT>(), UB = unit_bytes<QT>(), NC = 8 * NT, D = RING;
    extern __shared__ __align__(16) uint8_t s_x[];  // [2][cu][NT] fragment units, then the sums
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, i4 = lane & 3;
    const int ks = p.ks, part = (int)(blockIdx.x % ks);
    const int64_t tile = (int64_t)(blockIdx.x / ks) * GEMM_W + warp;
    const int64_t t0 = (int64_t)blockIdx.y * NC;
    const int ncol = (int)min((int64_t)NC, p.T - t0);
    const int ub = (int)(p.units * part / ks), ue = (int)(p.units * (part + 1) / ks);
    const bool live = tile < p.tiles;
    if (ks > 1) cluster_arrive();  // the others write into this CTA's shared memory when they know that it runs
    const uint8_t* wt = p.w + tile * p.units * UB;
    UnitRegs<QT> ring[D];
    if (live) {
#pragma unroll
        for (int d = 0; d < D; ++d)  // constant weights: before the wait
            if (ub + d < ue) ring[d].load(wt + (int64_t)(ub + d) * UB, lane);
    }
    pdl_wait();
    pdl_trigger();

    const uint8_t* xsrc = p.xf + (int64_t)blockIdx.y * p.units * (NT * XU);
    const uint32_t s_base = (uint32_t)__cvta_generic_to_shared(s_x);
    const int stage_bytes = p.cu * (NT * XU);
    auto stage = [&](int c) {
        const int b = ub + c * p.cu, e = min(ue, b + p.cu);
        const int n16 = max(0, e - b) * (NT * XU / 16);
        const uint32_t dst = s_base + (c & 1) * stage_bytes;
        const uint8_t* src = xsrc + (int64_t)b * (NT * XU);
        for (int i = tid; i < n16; i += GEMM_T) cp_async16(dst + i * 16, src + (int64_t)i * 16);
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    stage(0);
    uint64_t sum[NT][2];  // pairs of neighbouring columns, rows g and g + 8
#pragma unroll
    for (int n = 0; n < NT; ++n) sum[n][0] = sum[n][1] = 0;
    auto multiply = [&](const UnitRegs<QT>& w, const uint8_t* xu) {
        uint64_t dg[2][2];  // [block]{d, d} of rows g and g + 8
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int v = b ? w.d.y : w.d.x;
            const float2 d = __half22float2(*reinterpret_cast<const __half2*>(&v));
            dg[b][0] = pack2(d.x, d.x);
            dg[b][1] = pack2(d.y, d.y);
        }
        if constexpr (QT == PI_QT_Q8_0) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint4 xv = *reinterpret_cast<const uint4*>(xu + n * XU + lane * 16);
                const ulonglong2 dx = *reinterpret_cast<const ulonglong2*>(xu + n * XU + 512 + i4 * 16);
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    int s[4];
                    mma_s8(s, *reinterpret_cast<const uint4*>(&w.q[b]),
                           b ? make_uint2(xv.z, xv.w) : make_uint2(xv.x, xv.y));
                    const uint64_t d2 = b ? dx.y : dx.x;
                    sum[n][0] = fma2(pack2((float)s[0], (float)s[1]), mul2(dg[b][0], d2), sum[n][0]);
                    sum[n][1] = fma2(pack2((float)s[2], (float)s[3]), mul2(dg[b][1], d2), sum[n][1]);
                }
            }
        } else {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                uint32_t a[2][4];
                const uint32_t w0 = word(w.q[0], 2 * b), w1 = word(w.q[0], 2 * b + 1);
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    a[s][0] = nib_pair(w0, 2 * s);
                    a[s][1] = nib_pair(w1, 2 * s);
                    a[s][2] = nib_pair(w0, 2 * s + 1);
                    a[s][3] = nib_pair(w1, 2 * s + 1);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint8_t* xb = xu + n * XU + b * 1024 + lane * 16;
                    const uint4 x0 = *reinterpret_cast<const uint4*>(xb);
                    const uint4 x1 = *reinterpret_cast<const uint4*>(xb + 512);
                    float s[4] = {0.f, 0.f, 0.f, 0.f};
                    mma_f16(s, a[0], x0.z, x0.w);
                    mma_f16(s, a[1], x1.z, x1.w);
                    mma_f16(s, a[0], x0.x, x0.y);
                    mma_f16(s, a[1], x1.x, x1.y);
                    sum[n][0] = fma2(dg[b][0], pack2(s[0], s[1]), sum[n][0]);
                    sum[n][1] = fma2(dg[b][1], pack2(s[2], s[3]), sum[n][1]);
                }
            }
        }
    };
    for (int c = 0; c < p.nchunk; ++c) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();  // piece c has landed; nobody reads the other buffer any more
        if (c + 1 < p.nchunk) stage(c + 1);
        if (!live) continue;
        const uint8_t* xu = s_x + (c & 1) * stage_bytes;
        const int u0 = ub + c * p.cu, u1 = min(ue, u0 + p.cu);
        // a piece that is not the last has a multiple of D units, so unit u0 is in ring[0]
#pragma unroll 1
        for (int u = u0; u < u1; u += D, xu += D * NT * XU) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                if (u + d >= u1) break;
                multiply(ring[d], xu + d * NT * XU);
                if (u + d + D < ue) ring[d].load(wt + (int64_t)(u + d + D) * UB, lane);
            }
        }
    }
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const float2 u = unpack2(sum[n][0]), v = unpack2(sum[n][1]);
        acc[n][0] = u.x;
        acc[n][1] = u.y;
        acc[n][2] = v.x;
        acc[n][3] = v.y;
    }
    if (ks > 1) {  // n-tile n belongs to CTA n % ks of the cluster from here on: the parts go there
        cg::cluster_group cl = cg::this_cluster();
        float4* sums = reinterpret_cast<float4*>(s_x + p.sums) + warp * 32 + lane;  // [n / ks][part][warp][lane]
        cluster_wait();
        if (live) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
                cl.map_shared_rank(sums, n % ks)[((n / ks) * ks + part) * GEMM_T] =
                    make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
        }
        cluster_arrive();
        if (part >= NT) return;  // no n-tile is this CTA's
        cluster_wait();
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (n % ks != part) continue;
            float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int q = 0; q < ks; ++q) {
                const float4 v = sums[((n / ks) * ks + q) * GEMM_T];
                t.x += v.x;
                t.y += v.y;
                t.z += v.z;
                t.w += v.w;
            }
            acc[n][0] = t.x;
            acc[n][1] = t.y;
            acc[n][2] = t.z;
            acc[n][3] = t.w;
        }
    }
    if (!live) return;
    if (QT == PI_QT_Q4_0) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int u = n * 8 + 2 * i4;
            const float su = u < ncol ? p.xs[t0 + u] : 0.0f, sv = u + 1 < ncol ? p.xs[t0 + u + 1] : 0.0f;
            acc[n][0] *= su;
            acc[n][1] *= sv;
            acc[n][2] *= su;
            acc[n][3] *= sv;
        }
    }
    const int64_t row = tile * 16 + g;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        if (ks > 1 && n % ks != part) continue;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int col = n * 8 + 2 * i4 + e;
            if (col >= ncol) continue;
            float* y = p.y + (t0 + col) * p.n_out + row;
            if (row < p.n_out) y[0] = acc[n][e];
            if (row + 8 < p.n_out) y[8] = acc[n][2 + e];
        }
    }
}

// ---------------------------------------------------------------------------
// k_proj_adapters: y_t += B_a h_t. In a chunk of 64 tokens those of one adapter, up to eight
// together, are the columns of a product on the tensor cores (B exact in tf32 for f16 and
// bf16, two tf32 terms for f32; h in two terms: what the second terms leave, and the product of two
// second terms, is below 2^-21 of each product, as a few f32 roundings are); a warp's step is two tiles of 16 rows of one
// such group. A token is in one group only, so an adapter's NaN stays with its requests and
// every sum has one owner.
//
// A kernel of its own costs a second pass over y (mostly from L2), but its loads are as deep as
// the occupancy allows; in the epilogue of k_proj_gemm a warp went through the groups one memory
// latency after another (64 tokens, 2048 -> 151936, Q8_0, 16 adapters of rank 16: 224 us
// together, 167 apart, 130 without adapters; 16 tokens, 4096 -> 12288, Q4_0, rank 64: 35 / 30 /
// 21). Bound there: latency and issue (60%), 123 MB from memory in 40 us.
// ---------------------------------------------------------------------------
constexpr int AD_T = 256;
constexpr int AD_C = 64;  // tokens of a chunk
constexpr int AD_U = 2;   // tiles of a warp's step
constexpr int AD_CTAS = 3;  // of an SM; the grid is what runs at once, its warps stride over the steps

template <bool F32>
__global__ __launch_bounds__(AD_T, AD_CTAS) void k_proj_adapters(const LoraArgs L, const float* __restrict__ h, int64_t T,
                                                        int64_t n_out, int steps, float* __restrict__ y) {
    constexpr int ES = F32 ? 4 : 2;
    __shared__ int s_key[AD_C], s_tok[AD_C];
    __shared__ int4 s_group[AD_C];  // adapter, rank, first place in s_tok, tokens
    __shared__ int s_groups;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, i4 = lane & 3;
    const int64_t t0 = (int64_t)blockIdx.y * AD_C;
    const int ncol = (int)min((int64_t)AD_C, T - t0);
    // the kernels before this one have waited for what wrote the ids and weights before they let
    // it start: only y is waited for
    int rank = 0;
    if (tid < AD_C) s_key[tid] = tid < ncol ? lora_of(L, t0 + tid, &rank) : -1;
    __syncthreads();
    if (tid < AD_C) {
        const int a = rank > 0 ? s_key[tid] : -1;
        int less = 0, before = 0, all = 0;
        for (int q = 0; q < ncol; ++q) {
            const int k = s_key[q];
            less += k < a;
            all += k == a;
            before += k == a && q < tid;
        }
        const bool start = a >= 0 && (before & 7) == 0;
        if (a >= 0) s_tok[less + before] = tid;
        const uint32_t b = __ballot_sync(0xffffffffu, start);
        if (tid == 0) s_groups = __popc(b);
        asm volatile("bar.sync 1, 64;" ::: "memory");
        const int at = (warp ? s_groups : 0) + __popc(b & ((1u << lane) - 1u));
        asm volatile("bar.sync 1, 64;" ::: "memory");
        if (start) s_group[at] = make_int4(a, rank, less + before, min(8, all - before));
        if (tid == 32) s_groups += __popc(b);
    }
    __syncthreads();
    const int groups = s_groups, stride = (int)gridDim.x * (AD_T / 32);
    const bool f16 = L.dtype == PI_QT_F16;
    const int64_t row_bytes = (int64_t)L.R * ES;
    const uint8_t* bw = reinterpret_cast<const uint8_t*>(L.b) + 4 * i4 * ES;
    pdl_wait();
    pdl_trigger();
    int group = 0, step = (int)blockIdx.x * (AD_T / 32) + warp;
    while (true) {
        while (step >= steps && group < groups) {
            step -= steps;
            ++group;
        }
        if (group >= groups) break;
        const int64_t row0 = (int64_t)step * (16 * AD_U) + g;
        const int rows = (int)min(n_out - row0, (int64_t)(16 * AD_U));  // from row0 on; may be 0 or less
        const int4 gr = s_group[group];
        const float* hp = h + ((t0 + s_tok[gr.z + min(g, gr.w - 1)]) * L.R + 4 * i4) * 2;
        const uint8_t* b0 = bw + ((int64_t)gr.x * n_out + row0) * row_bytes;
        int64_t off[2 * AD_U];  // rows behind the last are not stored: they may hold the last one's
#pragma unroll
        for (int k = 0; k < 2 * AD_U; ++k) off[k] = min(8 * k, rows - 1) * row_bytes;
        float* yp[2];
        bool on[2];
        float old[2 * AD_U][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            on[e] = 2 * i4 + e < gr.w;
            yp[e] = y + (t0 + (on[e] ? s_tok[gr.z + 2 * i4 + e] : 0)) * n_out + row0;
#pragma unroll
            for (int k = 0; k < 2 * AD_U; ++k) old[k][e] = on[e] && 8 * k < rows ? yp[e][8 * k] : 0.0f;
        }
        float c[AD_U][4];
#pragma unroll
        for (int u = 0; u < AD_U; ++u) c[u][0] = c[u][1] = c[u][2] = c[u][3] = 0.0f;
#pragma unroll 1
        for (int r0 = 0; r0 < gr.y; r0 += 16) {
            const int left = gr.y - r0 - 4 * i4;  // rank entries of this lane's four that count
            float4 hl = make_float4(0.f, 0.f, 0.f, 0.f), hs = hl;  // large and small terms
            uint4 v[2 * AD_U];
#pragma unroll
            for (int k = 0; k < 2 * AD_U; ++k) v[k] = make_uint4(0, 0, 0, 0);
            if (left > 0) {
                hl = *reinterpret_cast<const float4*>(hp + r0 * 2);
                hs = *reinterpret_cast<const float4*>(hp + r0 * 2 + 4);
#pragma unroll
                for (int k = 0; k < 2 * AD_U; ++k) {
                    if constexpr (F32) {
                        const int4 w = ld_stream(b0 + off[k] + r0 * ES);
                        v[k] = make_uint4(w.x, w.y, w.z, w.w);
                    } else {
                        uint2 w;
                        asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];"
                                     : "=r"(w.x), "=r"(w.y)
                                     : "l"(b0 + off[k] + r0 * ES));
                        v[k].x = w.x;
                        v[k].y = w.y;
                    }
                }
            }
            uint32_t big[AD_U][2][4], small[AD_U][2][4];
#pragma unroll
            for (int k = 0; k < 2 * AD_U; ++k) {
                float f[4];
                if constexpr (F32) {
                    f[0] = __uint_as_float(v[k].x);
                    f[1] = __uint_as_float(v[k].y);
                    f[2] = __uint_as_float(v[k].z);
                    f[3] = __uint_as_float(v[k].w);
                } else if (f16) {
                    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v[k].x));
                    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&v[k].y));
                    f[0] = a.x;
                    f[1] = a.y;
                    f[2] = b.x;
                    f[3] = b.y;
                } else {
                    f[0] = __uint_as_float(v[k].x << 16);
                    f[1] = __uint_as_float(v[k].x & 0xffff0000u);
                    f[2] = __uint_as_float(v[k].y << 16);
                    f[3] = __uint_as_float(v[k].y & 0xffff0000u);
                }
                if (gr.y & 3) {  // the rank ends inside four entries; fours behind it were not loaded
#pragma unroll
                    for (int q = 1; q < 4; ++q)
                        if (q >= left) f[q] = 0.0f;
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) big[k >> 1][q >> 1][(k & 1) + 2 * (q & 1)] = __float_as_uint(f[q]);
            }
            const uint32_t h0 = __float_as_uint(hl.x), h1 = __float_as_uint(hl.y), h2 = __float_as_uint(hl.z),
                           h3 = __float_as_uint(hl.w);
#pragma unroll
            for (int u = 0; u < AD_U; ++u) {
                if constexpr (F32) {
#pragma unroll
                    for (int s = 0; s < 2; ++s)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const float f = __uint_as_float(big[u][s][q]);
                            big[u][s][q] = to_tf32(f);
                            small[u][s][q] = to_tf32(f - __uint_as_float(big[u][s][q]));
                        }
                    mma_tf32(c[u], small[u][0], h0, h1);
                    mma_tf32(c[u], small[u][1], h2, h3);
                }
                mma_tf32(c[u], big[u][0], __float_as_uint(hs.x), __float_as_uint(hs.y));
                mma_tf32(c[u], big[u][1], __float_as_uint(hs.z), __float_as_uint(hs.w));
                mma_tf32(c[u], big[u][0], h0, h1);
                mma_tf32(c[u], big[u][1], h2, h3);
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int k = 0; k < 2 * AD_U; ++k)
                if (on[e] && 8 * k < rows) yp[e][8 * k] = old[k][e] + c[k >> 1][(k & 1) * 2 + e];
        step += stride;
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
// n-tiles of 8 tokens are worked on in chunks of up to 8, as even as they come
int proj_chunk(int64_t T) {
    const int64_t ntt = (T + 7) / 8, chunks = (ntt + 7) / 8;
    return (int)((ntt + chunks - 1) / chunks);
}
ProjBufs proj_carve(const pi_proj* P, int64_t T, int64_t R, char* base) {
    PiBump b{base};
    ProjBufs o;
    const int64_t NT = proj_chunk(T), chunks = ((T + 7) / 8 + NT - 1) / NT;
    const int64_t xg = P->qtype == PI_QT_Q8_0 ? xunit_bytes<PI_QT_Q8_0>() : xunit_bytes<PI_QT_Q4_0>();
    o.xf = b.take<uint8_t>((size_t)(chunks * P->units * NT * xg));
    o.xs = b.take<float>((size_t)(P->qtype == PI_QT_Q4_0 ? T : 0));
    o.h = b.take<float>((size_t)(T * R) * 2);
    o.bytes = b.off + 256;
    return o;
}

template <int QT>
int proj_pack(pi_ctx* ctx, pi_proj* P, const uint8_t* raw, int src_on_host) {
    const int64_t nb = P->n_in / 32, row_bytes = proj_raw_bytes(QT, P->n_in), stride = P->units * unit_bytes<QT>();
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
        k_proj_pack<QT><<<(unsigned)(nt * P->units), 64>>>(src, nb, rows, P->units, P->w + t * stride);
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
    P->units = (n_in / 32 + 1) / 2;
    P->tiles = (n_out + 15) / 16;
    const int64_t ubytes = qtype == PI_QT_Q8_0 ? unit_bytes<PI_QT_Q8_0>() : unit_bytes<PI_QT_Q4_0>();
    if (P->tiles * P->units > INT32_MAX) {
        delete P;
        return pi_set_error(ctx, PI_ERR_ARG, "projection: too large");
    }
    int rc = PI_OK;
    if (pi_cuda_check(ctx, cudaMalloc((void**)&P->w, (size_t)(P->tiles * P->units * ubytes)), "cudaMalloc(projection)"))
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

// Parts of the blocks (ks) and stages. The time of a grid is about the rounds of CTAs that run at
// once times the units of a part plus what a CTA costs beside them (start, stage and join,
// about a dozen units' time). How many clusters run at once the runtime knows: clusters of
// three or five leave SMs of a GPC empty.
template <int QT, int NT>
pi_proj::Plan plan_gemm(const pi_proj* P, int64_t T, int64_t sms) {
    constexpr int XU = NT * xunit_bytes<QT>();
    const int64_t sets = (P->tiles + GEMM_W - 1) / GEMM_W, chunks = (T + 8 * NT - 1) / (8 * NT);
    auto kern = k_proj_gemm<QT, NT>;
    pi_smem_attr((const void*)kern, GEMM_SMEM);
    pi_proj::Plan best = {};
    int64_t least = INT64_MAX;
    for (int ks = 1; ks <= 8 && ks <= P->units; ++ks) {
        pi_proj::Plan q;
        q.ks = ks;
        // a part is staged whole where two CTAs of an SM have room for it beside the sums, in
        // pieces of a multiple of RING units otherwise
        const int64_t sums = ks > 1 ? (int64_t)((NT + ks - 1) / ks) * ks * GEMM_T * 16 : 0;
        const int64_t budget = 108 * 1024 - sums, part = (P->units + ks - 1) / ks;
        q.cu = (int)part;
        if (part * XU > budget) q.cu = (int)std::max<int64_t>(RING, budget / 2 / XU / RING * RING);
        q.nchunk = (int)((part + q.cu - 1) / q.cu);
        q.sums = std::min(q.nchunk, 2) * q.cu * XU;
        q.smem = (size_t)(q.sums + sums);
        if (q.smem > GEMM_SMEM) continue;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(sets * ks), (unsigned)chunks);
        cfg.blockDim = dim3(GEMM_T);
        cfg.dynamicSmemBytes = q.smem;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = (unsigned)ks;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        int clusters = 0;
        if (cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg) != cudaSuccess || clusters < 1) {
            cudaGetLastError();
            clusters = (int)(sms / ks);
        }
        const int64_t rounds = (sets * chunks + clusters - 1) / clusters, cost = rounds * (part + 12);
        if (cost < least) {
            least = cost;
            best = q;
        }
    }
    return best;
}

template <int QT, int NT>
cudaError_t launch_gemm(const pi_proj* P, ProjArgs a, int64_t sms, cudaStream_t st) {
    pi_proj::Plan q;
    {
        std::lock_guard<std::mutex> g(P->mu);
        const int64_t key = (a.T + 7) / 8;  // the plan goes by n-tiles
        auto it = P->plans.find(key);
        if (it == P->plans.end()) it = P->plans.emplace(key, plan_gemm<QT, NT>(P, a.T, sms)).first;
        q = it->second;
    }
    a.ks = q.ks;
    a.cu = q.cu;
    a.nchunk = q.nchunk;
    a.sums = q.sums;
    const int64_t sets = (a.tiles + GEMM_W - 1) / GEMM_W, chunks = (a.T + 8 * NT - 1) / (8 * NT);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(sets * a.ks), (unsigned)chunks);
    cfg.blockDim = dim3(GEMM_T);
    cfg.dynamicSmemBytes = q.smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)a.ks;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = a.ks > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, k_proj_gemm<QT, NT>, a);
}

template <int QT>
cudaError_t dispatch_gemm(const pi_proj* P, const ProjArgs& a, int NT, int64_t sms, cudaStream_t st) {
    switch (NT) {
        case 1: return launch_gemm<QT, 1>(P, a, sms, st);
        case 2: return launch_gemm<QT, 2>(P, a, sms, st);
        case 3: return launch_gemm<QT, 3>(P, a, sms, st);
        case 4: return launch_gemm<QT, 4>(P, a, sms, st);
        case 5: return launch_gemm<QT, 5>(P, a, sms, st);
        case 6: return launch_gemm<QT, 6>(P, a, sms, st);
        case 7: return launch_gemm<QT, 7>(P, a, sms, st);
        default: return launch_gemm<QT, 8>(P, a, sms, st);
    }
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
    const int NT = proj_chunk(T);
    {
        PiProfScope ps(ctx, st, "k_proj_prep");
        // the warps of a unit: many where there are few units (4 tokens, 11008 wide, rank 64: 29 us with
        // 4, 25 with 8, 23 with 16; 16 tokens, 4096: 30.4 / 29.2), few where there are many (231 tokens,
        // 640, rank 104: 71 with 4, 68 with 2), and none without 256 values of a row
        const int64_t units = T * (R / PREP_R);
        int S = units <= 128 ? 16 : (units <= 512 ? 8 : (units < 2048 ? 4 : 2));
        while (S > 2 && S * 128 >= P->n_in) S /= 2;
        const int64_t per = PREP_T / 32 / S, grid = T + (units + per - 1) / per;
        if (q8)
            pi_pdl_launch(k_proj_prep<PI_QT_Q8_0>, dim3((unsigned)grid), dim3(PREP_T), 0, st, x, T, P->n_in, P->units,
                          NT, B.xf, B.xs, L, B.h, S, ctx->dev_err);
        else
            pi_pdl_launch(k_proj_prep<PI_QT_Q4_0>, dim3((unsigned)grid), dim3(PREP_T), 0, st, x, T, P->n_in, P->units,
                          NT, B.xf, B.xs, L, B.h, S, ctx->dev_err);
    }
    {
        PiProfScope ps(ctx, st, "k_proj_gemm");
        const ProjArgs a{P->w, B.xf, B.xs, y, T, P->n_out, P->units, P->tiles, 1, 1, 1, 0};
        const int64_t sms = ctx->sm_count > 0 ? ctx->sm_count : 148;
        const cudaError_t e = q8 ? dispatch_gemm<PI_QT_Q8_0>(P, a, NT, sms, st) : dispatch_gemm<PI_QT_Q4_0>(P, a, NT, sms, st);
        if (e != cudaSuccess) return pi_cuda_check(ctx, e, "projection");
    }
    if (bank) {
        PiProfScope ps(ctx, st, "k_proj_adapters");
        const int64_t sms = ctx->sm_count > 0 ? ctx->sm_count : 148, steps = (P->n_out + 16 * AD_U - 1) / (16 * AD_U);
        const int64_t chunks = (T + AD_C - 1) / AD_C, most = std::min<int64_t>(T, AD_C) * steps;  // items of a chunk
        const int64_t ctas = std::min((most + AD_T / 32 - 1) / (AD_T / 32), std::max<int64_t>(1, AD_CTAS * sms / chunks));
        const dim3 grid((unsigned)ctas, (unsigned)chunks);
        if (L.dtype == PI_QT_F32)
            pi_pdl_launch(k_proj_adapters<true>, grid, dim3(AD_T), 0, st, L, B.h, T, P->n_out, (int)steps, y);
        else
            pi_pdl_launch(k_proj_adapters<false>, grid, dim3(AD_T), 0, st, L, B.h, T, P->n_out, (int)steps, y);
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
