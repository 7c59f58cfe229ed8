// Products of e4m3 matrices with a power-of-two scale for every row and every 128 entries of the summed axis, and the quantiser that makes
// such matrices: the Dense layer of ``mh_linear_bias_act_fwd`` (tf/blocks/mlp.py:275-280) with 8-bit operands.
//
//   quantise  e = the least integer with max |x| <= 448 2^e over a block; stored: e4m3(x 2^-e), ties to even, and the byte e + 127
//   product   C[m, n] = sum_b 2^(ea[m, b] + eb[n, b]) sum_{k in b} a[m, k] b[n, k]  (+ bias[n])
//
// A power of two as the scale makes x 2^-e exact, so a matrix is quantised to the same bits wherever it is done, and it is the form that the
// scaled matrix instruction takes beside its operands: the scales cost no vector instruction in the loop.  Both operands are stored with the
// summed axis contiguous and padded with zeros to whole blocks, so the loop has no tail in k.
#include "mh_lowp.h"

#include <atomic>
#include <type_traits>

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// ---- quantiser -----------------------------------------------------------------------------------------------------------------------
// The scale's exponent from the bits of the block's largest magnitude: amax = 1.f 2^(E - 127) <= 448 2^e = 1.75 2^(8 + e) for e = E - 135, one more where
// 1.f > 1.75.  -126 below keeps 2^e and 2^-e normal numbers.
__device__ __forceinline__ int q_exponent(uint32_t b) {
    if (b == 0) return 0;
    const int e = (int)(b >> 23) - 135 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < -126 ? -126 : e;
}
__device__ __forceinline__ float q_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// An infinity or NaN becomes NaN in e4m3 and leaves its block's scale to the others.  Magnitudes are compared as bits, an AND and half a three-way
// maximum each, and whether a wavefront holds such a value is seen from the largest: only then are they looked at one by one (q_clean first, with
// which the conversion needs no care for them, then q_bits<true>).
constexpr uint32_t Q_INF = 0x7f800000u;
template <bool ODD>
__device__ __forceinline__ uint32_t q_bits(float v) {
    const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
    return ODD && b >= Q_INF ? 0u : b;
}
__device__ __forceinline__ uint32_t q_max(uint32_t a, uint32_t b) { return a > b ? a : b; }
template <bool ODD, int N>
__device__ __forceinline__ uint32_t q_most(const float (&v)[N]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = q_max(m, q_bits<ODD>(v[i]));
    return m;
}
template <int N>
__device__ __forceinline__ void q_clean(float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = q_bits<false>(v[i]) >= Q_INF ? __uint_as_float(0x7fc00000u) : v[i];
}
__device__ __forceinline__ uint32_t q_pack4(float a, float b, float c, float d) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// Blocks along the rows of x.  A wavefront takes four blocks (512 entries, 8 a lane: 16 lanes share a block) of one row and writes one word of
// scales; one pass, bound by its reads and writes: 65536 x 3341 fp32 201 us, 5.5 TB/s; 65536 x 512 25 us, 6.8 TB/s
// (medians of a trace, as all kernel times in this file that are not set against another).
template <typename T>
__global__ __launch_bounds__(256) void fp8_quantize_rows_kernel(const T* __restrict__ x, int64_t ldx, int64_t R, int K, int quads, uint8_t* __restrict__ q,
                                                               int64_t ldq, uint8_t* __restrict__ s, int64_t lds) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)(blockIdx.x / (uint32_t)quads) * 4 + (threadIdx.x >> 6);
    const int quad = (int)(blockIdx.x % (uint32_t)quads);
    if (row >= R) return;
    const int k = quad * 512 + lane * 8;
    float v[8];
    const T* p = x + row * ldx + k;
    if (k + 8 <= K) {
        lp_load8(p, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = k + i < K ? lp_float(p[i]) : 0.f;
    }
    uint32_t a = q_most<false>(v);
    if (__any(a >= Q_INF)) {
        q_clean(v);
        a = q_most<true>(v);
    }
#pragma unroll
    for (int m = 8; m; m >>= 1) a = q_max(a, __shfl_xor(a, m));
    const int e = q_exponent(a);
    const float inv = q_pow2(-e);
    const int kp = (K + 127) / 128 * 128;
    if (k < kp) {
        uint2 w;
        w.x = q_pack4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
        w.y = q_pack4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
        *reinterpret_cast<uint2*>(q + row * ldq + k) = w;
    }
    uint32_t sw = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) sw |= (uint32_t)(__shfl(e, 16 * b) + 127) << (8 * b);
    if (lane == 0) *reinterpret_cast<uint32_t*>(s + row * lds + quad * 4) = sw;
}

// Blocks along the columns of x: qt[c, r] = x[r, c], and with ROWS those along its rows from the same read.  A workgroup takes 128 x 128; a lane holds
// eight rows of four columns.  The rows' maxima meet by halves -- 4, 2, 1 values, then two more steps -- which leaves row i's with lanes 4 i to
// 4 i + 3 of its half wavefront; the columns' meet in LDS.  The tile turns round in LDS so that eight lanes write one 128-byte line of qt; sixteen
// bytes chunk h of column c lie at h ^ ((c >> 2) & 7), or all 32 lanes of a write would meet in two banks.  colsum, if given, receives the tile's column
// sums ([blocks, C]).  Bound by memory: 65536 x 512 fp32 26 us, 6.4 TB/s, and 34 us with ROWS (6.0 TB/s; the two forms apart 50); 65536 x 3341, whose rows
// start at any word, 233 us, 4.7 TB/s.  Single columns in place of four neighbouring ones a lane took 26 us for 16384 x 1024, 16 now; the order of the
// tiles made no difference.
template <typename T, bool ROWS>
__global__ __launch_bounds__(512) void fp8_quantize_tiles_kernel(const T* __restrict__ x, int64_t ldx, int64_t R, int64_t C, int cblocks, int rblocks,
                                                                uint8_t* __restrict__ q, int64_t ldq, uint8_t* __restrict__ s, int64_t lds,
                                                                uint8_t* __restrict__ qt, int64_t ldqt, uint8_t* __restrict__ st, int64_t ldst,
                                                                float* __restrict__ colsum) {
    __shared__ __attribute__((aligned(16))) uint32_t most[8][128];
    __shared__ __attribute__((aligned(16))) float sums[8][128];
    __shared__ __attribute__((aligned(16))) uint8_t tile[128][128];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, half = lane >> 5, c4 = (lane & 31) * 4;
    const int cb = (int)(blockIdx.x % (uint32_t)cblocks), rb = (int)(blockIdx.x / (uint32_t)cblocks);
    const int64_t c = (int64_t)cb * 128 + c4, r0 = (int64_t)rb * 128 + w * 16 + half * 8;
    float v[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const T* p = x + (r0 + i) * ldx + c;
        if (r0 + i < R && c + 4 <= C) {
            lp_load4(p, v[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i][j] = r0 + i < R && c + j < C ? lp_float(p[j]) : 0.f;
        }
    }
    if (colsum) {
        f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) t[j] += v[i][j];
#pragma unroll
        for (int j = 0; j < 4; ++j) t[j] += __shfl_xor(t[j], 32);
        if (half == 0) *reinterpret_cast<f32x4*>(&sums[w][c4]) = t;
    }
    uint32_t a[4] = {0, 0, 0, 0}, m[8];
    auto maxima = [&](auto odd) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            m[i] = q_most<decltype(odd)::value>(v[i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) a[j] = q_max(i ? a[j] : 0, q_bits<decltype(odd)::value>(v[i][j]));
        }
    };
    maxima(std::false_type{});
    if (__any(q_max(q_max(a[0], a[1]), q_max(a[2], a[3])) >= Q_INF)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) q_clean(v[i]);
        maxima(std::true_type{});
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = q_max(a[j], __shfl_xor(a[j], 32));
    if (half == 0) *reinterpret_cast<uint4*>(&most[w][c4]) = make_uint4(a[0], a[1], a[2], a[3]);
    if (ROWS) {
#pragma unroll
        for (int n = 4; n; n >>= 1)
#pragma unroll
            for (int i = 0; i < n; ++i) {
                const bool up = lane & (4 * n);
                const uint32_t keep = up ? m[n + i] : m[i], give = up ? m[i] : m[n + i];
                m[i] = q_max(keep, __shfl_xor(give, 4 * n));
            }
        m[0] = q_max(m[0], __shfl_xor(m[0], 2));
        m[0] = q_max(m[0], __shfl_xor(m[0], 1));
        const int e = q_exponent(m[0]), mine = (lane >> 2) & 7;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float inv = q_pow2(-__shfl(e, (lane & 32) + 4 * i));
            if (r0 + i < R) *reinterpret_cast<uint32_t*>(q + (r0 + i) * ldq + c) = q_pack4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
        }
        if ((lane & 3) == 0 && r0 + mine < R) {
            s[(r0 + mine) * lds + cb] = (uint8_t)(e + 127);
            if (cb == cblocks - 1)
                for (int b = cblocks; b & 3; ++b) s[(r0 + mine) * lds + b] = 127;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint4 o = *reinterpret_cast<const uint4*>(&most[i][c4]);
        a[0] = q_max(a[0], o.x), a[1] = q_max(a[1], o.y), a[2] = q_max(a[2], o.z), a[3] = q_max(a[3], o.w);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int e = q_exponent(a[j]);
        const float inv = q_pow2(-e);
        uint2 o;
        o.x = q_pack4(v[0][j] * inv, v[1][j] * inv, v[2][j] * inv, v[3][j] * inv);
        o.y = q_pack4(v[4][j] * inv, v[5][j] * inv, v[6][j] * inv, v[7][j] * inv);
        *reinterpret_cast<uint2*>(&tile[c4 + j][((w ^ (lane & 7)) << 4) + half * 8]) = o;
        if (w == 0 && half == 0 && c + j < C) {
            st[(c + j) * ldst + rb] = (uint8_t)(e + 127);
            if (rb == rblocks - 1)
                for (int b = rblocks; b & 3; ++b) st[(c + j) * ldst + b] = 127;
        }
    }
    if (colsum && threadIdx.x < 128 && (int64_t)cb * 128 + threadIdx.x < C) {
        float u = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) u += sums[i][threadIdx.x];
        colsum[(int64_t)rb * C + cb * 128 + threadIdx.x] = u;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int col = i * 64 + threadIdx.x / 8, h = threadIdx.x & 7;
        const int64_t cc = (int64_t)cb * 128 + col;
        if (cc < C) *reinterpret_cast<uint4*>(qt + cc * ldqt + (int64_t)rb * 128 + h * 16) = *reinterpret_cast<const uint4*>(&tile[col][(h ^ ((col >> 2) & 7)) << 4]);
    }
}

// out[c] = sum_b part[b, c]: sixteen wavefronts take every sixteenth b of 64 columns, then their sums in order
__global__ __launch_bounds__(1024) void fp8_colsum_kernel(const float* __restrict__ part, int blocks, int64_t C, float* __restrict__ out) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    float t = 0.f;
    if (c < C) {
#pragma unroll 8
        for (int b = w; b < blocks; b += 16) t += part[(int64_t)b * C + c];
    }
    red[w][lane] = t;
    __syncthreads();
    if (w || c >= C) return;
    t = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += red[i][lane];
    out[c] = t;
}

// ---- product -------------------------------------------------------------------------------------------------------------------------
struct F8Args {
    const uint8_t *a, *as, *b, *bs;
    int64_t lda, ldas, ldb, ldbs;
    int64_t M, N;
    int kblocks, kb_split;  // blocks of 128 in all, and in each slice of blockIdx.y (a multiple of 4)
    int mt, nt, per_xcd;    // output tiles, and how many of them an XCD takes
    const float* bias;
    int kind;  // MH_F32 / MH_BF16 / MH_F16
    void* out;
    int64_t ldo, slab;  // slab: entries between the slices' partial outputs
    int vec;            // entries of an output row that can be stored together: 1: four, 2: eight of 16 bits as well, 0: each alone
};

__device__ __forceinline__ void f8_dma16(const void* g, void* l) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g, (__attribute__((address_space(3))) void*)l, 16, 0, 0);
}
__device__ __forceinline__ void f8_dma4(const void* g, void* l) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g, (__attribute__((address_space(3))) void*)l, 4, 0, 0);
}

// 32 e4m3 of one row, scaled, as four operands of the bf16 matrix instruction: e4m3 has 4 significant bits and bf16 8, so nothing is lost
__device__ __forceinline__ void f8_widen(const i32x8& v, float scale, bf16x8 (&o)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const bf16x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * j], scale, false), p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * j], scale, true);
        const bf16x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * j + 1], scale, false), p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * j + 1], scale, true);
        o[j] = bf16x8{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
    }
}

__device__ __forceinline__ void f8_store4(const F8Args& g, int64_t m, int64_t n, float v0, float v1, float v2, float v3, int64_t slab) {
    const int64_t at = slab + m * g.ldo + n;
    const float v[4] = {v0, v1, v2, v3};
    if (g.vec && n + 4 <= g.N) {
        if (g.kind == MH_F32) {
            *reinterpret_cast<f32x4*>(static_cast<float*>(g.out) + at) = f32x4{v0, v1, v2, v3};
        } else {
            uint2 w;
            w.x = g.kind == MH_BF16 ? lp_pack_bf16(v0, v1) : lp_pack_f16(v0, v1);
            w.y = g.kind == MH_BF16 ? lp_pack_bf16(v2, v3) : lp_pack_f16(v2, v3);
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(g.out) + at) = w;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n + i < g.N) {
            if (g.kind == MH_F32) static_cast<float*>(g.out)[at + i] = v[i];
            else static_cast<uint16_t*>(g.out)[at + i] = (uint16_t)(g.kind == MH_BF16 ? lp_pack_bf16(v[i], 0.f) : lp_pack_f16(v[i], 0.f));
        }
}

// eight entries of a row in 16 bits
__device__ __forceinline__ void f8_store8(const F8Args& g, int64_t m, int64_t n, const f32x4& lo, const f32x4& hi, const float (&b)[8], int64_t slab) {
    const int64_t at = slab + m * g.ldo + n;
    uint16_t* o = static_cast<uint16_t*>(g.out) + at;
    const float v[8] = {lo[0] + b[0], lo[1] + b[1], lo[2] + b[2], lo[3] + b[3], hi[0] + b[4], hi[1] + b[5], hi[2] + b[6], hi[3] + b[7]};
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = g.kind == MH_BF16 ? lp_pack_bf16(v[2 * i], v[2 * i + 1]) : lp_pack_f16(v[2 * i], v[2 * i + 1]);
    if (g.vec > 1 && n + 8 <= g.N) {
        *reinterpret_cast<uint4*>(o) = make_uint4(w[0], w[1], w[2], w[3]);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (n + i < g.N) o[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
}
// LDS written before is read after, by the same wavefront
__device__ __forceinline__ void f8_wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Tiled product.  WIDE: operands widened to bf16 on the way from LDS, for outputs of fp32 and fp16.  The 8-bit matrix instruction takes its
// products in groups of eight and cuts each at 2^-13 of the group's largest (measured with single products on both shapes; the groups' sums
// are then added in fp32): at most 7 2^-13 = 2^-10.2 of sum |a b|, 1.5e-5 of the norm on random values.  A bf16 output takes it all the same, for twice
// the rate: where the terms do not cancel its rounding, 2^-8 of the result, is larger, but where they do the sum can be off by many of its steps (quantising
// the operands is off by up to 2^-4 of each term already).  The finer types take the bf16 instruction, which adds in fp32, at half the rate.
// Each wavefront holds (BM / WM) x (BN / WN) of the output as 32 x 32 accumulators, rows of b as the instruction's rows: a lane then owns four
// neighbouring columns of C.  Tiles of one block of k (128 bytes a row) come by direct-to-LDS loads, two stages, one barrier a block; 16-byte
// chunk c of row r lies at c ^ ((r >> 1) & 7), which spreads the 16 rows of a read phase over all 64 banks.  Bound by the matrix pipe: 8192^3 463 us (440 at
// best), 2380 TFLOP/s, and WIDE 809 us, 1360 TFLOP/s; 65536 x 512 x 3341 WIDE 226 us right behind the quantiser (185 at best), 990 TFLOP/s.
template <int BM, int BN, int WM, int WN, bool WIDE>
__global__ __launch_bounds__(WM * WN * 64, 2) void fp8_gemm_kernel(const F8Args g) {
    constexpr int NT = WM * WN * 64, TM = BM / WM / 32, TN = BN / WN / 32;
    constexpr int STAGE = (BM + BN) * 128, DMA = STAGE / 16 / NT, SCALES = (BM + BN) * 4, SDMA = SCALES / 4 / NT;
    static_assert(SDMA * NT * 4 == SCALES && DMA * NT * 16 == STAGE, "every thread issues the same number of loads");
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, l31 = lane & 31, h = lane >> 5;
    const int wm = wave / WN, wn = wave % WN;
    // tile of this workgroup: consecutive workgroups go to the eight XCDs in turn, so each XCD takes a run of tiles of its own, in groups of
    // eight tile rows: the tiles in flight on one L2 share their operands' panels
    const int tile = (int)(blockIdx.x & 7) * g.per_xcd + (int)(blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= g.per_xcd || tile >= g.mt * g.nt) return;
    const int group = tile / (8 * g.nt), in = tile - group * 8 * g.nt, rows = g.mt - group * 8 < 8 ? g.mt - group * 8 : 8;
    const int64_t m0 = (int64_t)(group * 8 + in % rows) * BM, n0 = (int64_t)(in / rows) * BN;
    const int kb0 = blockIdx.y * g.kb_split, kb1 = kb0 + g.kb_split < g.kblocks ? kb0 + g.kb_split : g.kblocks;

    // sources of this thread's loads as 32-bit offsets from the tile's first rows (rows past the end repeat the last: never stored)
    const uint8_t *const ta = g.a + m0 * g.lda, *const tb = g.b + n0 * g.ldb, *const tas = g.as + m0 * g.ldas, *const tbs = g.bs + n0 * g.ldbs;
    const int ma = g.M - m0 < BM ? (int)(g.M - m0) - 1 : BM - 1, nb = g.N - n0 < BN ? (int)(g.N - n0) - 1 : BN - 1;
    constexpr int DA = BM * 8 / NT;
    uint32_t src[DMA];
#pragma unroll
    for (int j = 0; j < DMA; ++j) {
        const int L = (j < DA ? j : j - DA) * NT + threadIdx.x, r = L >> 3, c = (L & 7) ^ ((r >> 1) & 7);
        src[j] = j < DA ? (uint32_t)((r < ma ? r : ma) * g.lda) + c * 16 : (uint32_t)((r < nb ? r : nb) * g.ldb) + c * 16;
    }
    uint8_t* const sbase = smem + 2 * STAGE;
    auto issue = [&](int kb, int stage) {
        uint8_t* st = smem + (stage & 1) * STAGE;
        const uint8_t *pa = ta + (int64_t)kb * 128, *pb = tb + (int64_t)kb * 128;
#pragma unroll
        for (int j = 0; j < DMA; ++j) f8_dma16((j < DA ? pa : pb) + src[j], st + (j * NT + wave * 64) * 16);
    };
    auto issue_scales = [&](int kb, int group) {  // of four blocks, one word a row
#pragma unroll
        for (int j = 0; j < SDMA; ++j) {
            const int r = j * NT + threadIdx.x;
            const uint8_t* p = r < BM ? tas + (r < ma ? r : ma) * g.ldas : tbs + (r - BM < nb ? r - BM : nb) * g.ldbs;
            f8_dma4(p + (kb & ~3), sbase + (group & 1) * SCALES + (j * NT + wave * 64) * 4);
        }
    };
    f32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    // where this lane's fragments lie in a stage: its row, and in it the two chunks of each half of the block
    const int arow = (wm * (BM / WM) + l31) * 128, brow = (BM + wn * (BN / WN) + l31) * 128, sw = (l31 >> 1) & 7;
    const int chunk[2][2] = {{((2 * h) ^ sw) << 4, ((2 * h + 1) ^ sw) << 4}, {((4 + 2 * h) ^ sw) << 4, ((5 + 2 * h) ^ sw) << 4}};
    auto read = [&](int kb, int half, int row) {
        const uint8_t* st = smem + (kb & 1) * STAGE + row;
        const i32x4 x = *reinterpret_cast<const i32x4*>(st + chunk[half][0]);
        const i32x4 y = *reinterpret_cast<const i32x4*>(st + chunk[half][1]);
        return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    int sa[TM], sb[TN], ta_[TM], tb_[TN];
    auto read_scales = [&](int kb, int (&x)[TM], int (&y)[TN]) {
        const uint8_t* sp = sbase + ((kb >> 2) & 1) * SCALES + (kb & 3);
#pragma unroll
        for (int i = 0; i < TM; ++i) x[i] = sp[arow / 32 + i * 128];
#pragma unroll
        for (int j = 0; j < TN; ++j) y[j] = sp[brow / 32 + j * 128];
    };
    // A block is 2 TM steps: a step multiplies one 32-row fragment of a with the TN fragments of b, over half of the block.  a's fragments
    // are read two steps ahead into a ring of four, b's for the next half within the half before.  The barrier of a block lies two steps
    // before the end of the block before it, so the matrix pipe has work on both sides of it.
    constexpr int S = 2 * TM;
    i32x8 fa[4], fb[2][TN];
    bf16x8 wb[TN][4];
    auto widen_b = [&](int half) {
        if (WIDE) {
#pragma unroll
            for (int j = 0; j < TN; ++j) f8_widen(fb[half][j], __uint_as_float((uint32_t)sb[j] << 23), wb[j]);
        }
    };
    auto multiply = [&](int step) {
        const int i = step % TM, half = step / TM;
        if (!WIDE) {
#pragma unroll
            for (int j = 0; j < TN; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[half][j], fa[step & 3], acc[i][j], 0, 0, 0, sb[j], 0, sa[i]);
        } else {
            bf16x8 wa[4];
            f8_widen(fa[step & 3], __uint_as_float((uint32_t)sa[i] << 23), wa);
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[j][q], wa[q], acc[i][j], 0, 0, 0);
        }
    };
    issue_scales(kb0, kb0 >> 2);
    issue(kb0, kb0);
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    issue(kb0 + 1 < kb1 ? kb0 + 1 : kb0, kb0 + 1);
    read_scales(kb0, sa, sb);
#pragma unroll
    for (int j = 0; j < TN; ++j) fb[0][j] = read(kb0, 0, brow + j * 4096);
    fa[0] = read(kb0, 0, arow);
    fa[1] = read(kb0, 0, arow + 4096);
    // No branch in the body, or the compiler moves the multiplications behind the barrier: past the end the loads repeat the last block, into
    // the stage that would have been its turn, and what is read of it is not used.
    auto body = [&](int kb, bool scales) {
        const int one = kb + 1, two = kb + 2 < kb1 ? kb + 2 : kb1 - 1;
#pragma unroll
        for (int step = 0; step < S; ++step) {
            if (step == S - 2) {
                // block kb + 1 has arrived, and every wavefront holds what it still needs of block kb
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                if (scales) issue_scales(two, (kb + 2) >> 2);
                issue(two, kb);
                read_scales(one, ta_, tb_);
#pragma unroll
                for (int j = 0; j < TN; ++j) fb[0][j] = read(one, 0, brow + j * 4096);
            }
            if (step + 2 < S) fa[(step + 2) & 3] = read(kb, (step + 2) / TM, arow + (step + 2) % TM * 4096);
            else fa[(step + 2) & 3] = read(one, 0, arow + (step + 2 - S) * 4096);
            if (step == TM - 2) {
#pragma unroll
                for (int j = 0; j < TN; ++j) fb[1][j] = read(kb, 1, brow + j * 4096);
            }
            if (step % TM == 0) widen_b(step / TM);
            multiply(step);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) sa[i] = ta_[i];
#pragma unroll
        for (int j = 0; j < TN; ++j) sb[j] = tb_[j];
    };
    int kb = kb0;
    for (; kb + 4 <= kb1; kb += 4) {
        body(kb, false);
        body(kb + 1, false);
        body(kb + 2, true);  // the next four blocks' scales, beside the first of them
        body(kb + 3, false);
    }
    for (; kb < kb1; ++kb) body(kb, false);
    // Output: acc[i][j][4 q + e] = C[m0 + .. + 32 i + l31][n0 + .. + 32 j + 8 q + 4 h + e].  A wavefront turns 32 rows round in LDS and stores whole
    // stretches of rows (stored from the accumulators, eight or sixteen bytes of 32 rows at a time, 1000 x 50000 x 128 took 62 us).
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the last repeated loads
    __syncthreads();
    constexpr int CW = BN / WN, PITCH = CW + 4;
    static_assert(WM * WN * 32 * PITCH * 4 <= 2 * STAGE, "the turned rows fit the stages");
    float* const buf = reinterpret_cast<float*>(smem) + wave * 32 * PITCH;
    const int64_t nw = n0 + wn * CW, mw = m0 + wm * (BM / WM), slab = (int64_t)blockIdx.y * g.slab;
    const bool wide_out = g.kind == MH_F32;
    const int per = wide_out ? 4 : 8, lpr = CW / per, c = lane % lpr * per;  // entries a lane stores, lanes a row, this lane's column
    float bias[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) bias[e] = g.bias && e < per && nw + c + e < g.N ? g.bias[nw + c + e] : 0.f;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<f32x4*>(buf + l31 * PITCH + j * 32 + 8 * q + 4 * h) =
                    f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        f8_wave_fence();
        for (int r = lane / lpr; r < 32; r += 64 / lpr) {
            const int64_t m = mw + i * 32 + r;
            if (m >= g.M) break;
            const f32x4 lo = *reinterpret_cast<const f32x4*>(buf + r * PITCH + c);
            if (wide_out) {
                f8_store4(g, m, nw + c, lo[0] + bias[0], lo[1] + bias[1], lo[2] + bias[2], lo[3] + bias[3], slab);
            } else {
                const f32x4 hi = *reinterpret_cast<const f32x4*>(buf + r * PITCH + c + 4);
                f8_store8(g, m, nw + c, lo, hi, bias, slab);
            }
        }
        f8_wave_fence();
    }
}

// 32 entries as 8-bit values and their scale's byte: the quantiser's own rule, the four lanes that share a block and a row agreeing on it
__device__ __forceinline__ i32x8 f8_quantize32(float (&v)[32], uint32_t& scale) {
    uint32_t a = q_most<false>(v);
    if (__any(a >= Q_INF)) {
        q_clean(v);
        a = q_most<true>(v);
    }
    a = q_max(a, __shfl_xor(a, 16));
    a = q_max(a, __shfl_xor(a, 32));
    const int e = q_exponent(a);
    const float inv = q_pow2(-e);
    scale = (uint32_t)(e + 127);
    i32x8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (int)q_pack4(v[4 * i] * inv, v[4 * i + 1] * inv, v[4 * i + 2] * inv, v[4 * i + 3] * inv);
    return r;
}
struct f8_stored {};  // in place of an element type: a is in its 8-bit form

// What a lane holds of a row of a for one block of k: its 32 entries in the 8-bit form, or as they come.
template <typename X>
struct F8Lane {
    static constexpr int N = sizeof(X) * 2;  // 16-byte vectors
    uint4 w[N];
    __device__ __forceinline__ void load(const X* p, int left) {
        if (left >= 32) {
#pragma unroll
            for (int i = 0; i < N; ++i) w[i] = lp_load16(p + i * lp_vec<X>::N);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                X v[lp_vec<X>::N] = {};
#pragma unroll
                for (int j = 0; j < lp_vec<X>::N; ++j)
                    if (i * lp_vec<X>::N + j < left) v[j] = p[i * lp_vec<X>::N + j];
                __builtin_memcpy(&w[i], v, 16);
            }
        }
    }
    __device__ __forceinline__ i32x8 values(uint32_t& scale) const {
        float v[32];
        const X* type = nullptr;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float u[lp_vec<X>::N];
            lp_unpack(w[i], u, type);
#pragma unroll
            for (int j = 0; j < lp_vec<X>::N; ++j) v[i * lp_vec<X>::N + j] = u[j];
        }
        return f8_quantize32(v, scale);
    }
};
template <>
struct F8Lane<f8_stored> {
    i32x4 lo, hi;
    uint32_t s;
    __device__ __forceinline__ void load(const uint8_t* p, const uint8_t* ps) {
        lo = *reinterpret_cast<const i32x4*>(p);
        hi = *reinterpret_cast<const i32x4*>(p + 16);
        s = *ps;
    }
    __device__ __forceinline__ i32x8 values(uint32_t& scale) const {
        scale = s;
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

// Few rows of a (at most 16 MT): bound by reading b once.  A wavefront takes 16 NB rows of b for the 16 x 16 x 128 instruction; of a workgroup's eight,
// WK share the blocks of k and the others have rows of their own.  The instruction wants 16 rows in neighbouring lanes, which as loads would ask the
// cache for a line 16 bytes at a time (48 x 4096 -> 14341 took 28 us so): b comes by direct-to-LDS loads of whole lines into two stages of the
// wavefront's own, the next block's while one is multiplied, and no barrier is needed.  Partial sums meet in LDS in a fixed order and leave as
// whole stretches of output rows.  X: the type of a where it is quantised on the way (at most 16 rows: the work is done again for every 16 NB
// rows of b), or f8_stored.
// 16 x 4096 -> 65536 45 us, 6.1 TB/s; 48 x 4096 -> 14341 20 us, 3.0 TB/s (225 workgroups, one round, and the word of b's scales is asked for behind the next
// block's lines, so that its use waits for those too: the two stages overlap between wavefronts, not within one); 1 x 1024 -> 4096 4.8 us, nearly all of it
// a launch.
constexpr int RW = 8;  // wavefronts
template <int NB>
constexpr int f8_rows_stage() {
    return NB * 16 * 128;
}
template <int MT, int NB, bool WIDE, typename X>
__global__ __launch_bounds__(64 * RW, 2) void fp8_rows_kernel(const F8Args g, const X* __restrict__ x, int64_t ldx, int K, int wk) {
    constexpr bool STORED = std::is_same<X, f8_stored>::value;
    constexpr int PITCH = NB * 16 + 4, STAGE = f8_rows_stage<NB>();
    static_assert(16 * PITCH * 4 <= 2 * STAGE, "a wavefront's partial sums fit its stages");
    extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, l15 = lane & 15, h = lane >> 4;
    const int wn = RW / wk;  // row groups of the workgroup
    const int64_t nblock = (int64_t)blockIdx.x * wn * (16 * NB), n0 = nblock + wave / wk * (16 * NB);
    // this wavefront's blocks of k: whole words of scales where there are enough
    int share = (g.kblocks + wk - 1) / wk;
    if (share >= 4) share = (share + 3) & ~3;
    const int kb0 = wave % wk * share, kb1 = kb0 + share < g.kblocks ? kb0 + share : g.kblocks;
    uint8_t* const stage = smem + wave * 2 * STAGE;
    const int64_t nf = n0 < g.N ? n0 : g.N - 1;  // a group past the end reads the last row and stores nothing
    const uint8_t *const tb = g.b + nf * g.ldb, *const tbs = g.bs + nf * g.ldbs;
    const int last = g.N - nf < 16 * NB ? (int)(g.N - nf) - 1 : 16 * NB - 1;
    uint32_t src[2 * NB], ssrc[NB];
#pragma unroll
    for (int j = 0; j < 2 * NB; ++j) {
        const int r = 8 * j + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
        src[j] = (uint32_t)((r < last ? r : last) * g.ldb) + c * 16;
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) ssrc[j] = (uint32_t)((16 * j + l15 < last ? 16 * j + l15 : last) * g.ldbs);
    auto issue = [&](int kb) {
#pragma unroll
        for (int j = 0; j < 2 * NB; ++j) f8_dma16(tb + (int64_t)kb * 128 + src[j], stage + (kb & 1) * STAGE + j * 1024);
        asm volatile("" ::: "memory");  // all of b's lines first, then a: mixed by the compiler, 48 x 4096 -> 14341 took 19.9 us instead of 19.2
        __builtin_amdgcn_sched_barrier(0);
    };
    const uint8_t *pa[MT], *psa[MT];
    const X* px[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t m = 16 * i + l15 < g.M ? 16 * i + l15 : g.M - 1;
        if constexpr (STORED) {
            pa[i] = g.a + m * g.lda + h * 32;
            psa[i] = g.as + m * g.ldas;
        } else {
            px[i] = x + m * ldx + h * 32;
        }
    }
    f32x4 acc[MT][NB];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    uint32_t sb[NB];
    struct Block {
        F8Lane<X> a[MT];
    };
    auto load = [&](int kb, Block& v) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            if constexpr (STORED) v.a[i].load(pa[i] + (int64_t)kb * 128, psa[i] + kb);
            else v.a[i].load(px[i] + (int64_t)kb * 128, K - kb * 128 - h * 32);
        }
    };
    // Loads arrive in order: with no more left on the way than the next block's lines of b, which were asked for after this block's, those are there.
    auto multiply = [&](int kb, Block& v) {
        if (kb == kb0 || (kb & 3) == 0) {
#pragma unroll
            for (int j = 0; j < NB; ++j) sb[j] = *reinterpret_cast<const uint32_t*>(tbs + (kb & ~3) + ssrc[j]);
        }
        if (kb + 1 < kb1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NB) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const uint8_t* st = stage + (kb & 1) * STAGE;
        const int sw = (l15 >> 1) & 7, sh = (kb & 3) * 8;
        i32x8 va[MT];
        uint32_t sa[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) va[i] = v.a[i].values(sa[i]);
        bf16x8 wa[MT][4];
        if (WIDE) {
#pragma unroll
            for (int i = 0; i < MT; ++i) f8_widen(va[i], __uint_as_float(sa[i] << 23), wa[i]);
        }
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const i32x4 lo = *reinterpret_cast<const i32x4*>(st + (16 * j + l15) * 128 + (((2 * h) ^ sw) << 4));
            const i32x4 hi = *reinterpret_cast<const i32x4*>(st + (16 * j + l15) * 128 + (((2 * h + 1) ^ sw) << 4));
            const i32x8 vb = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            const uint32_t s = sb[j] >> sh;
            if (!WIDE) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(vb, va[i], acc[i][j], 0, 0, 0, (int)s, 0, (int)sa[i]);
            } else {
                bf16x8 wb[4];
                f8_widen(vb, __uint_as_float((s & 255u) << 23), wb);
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int i = 0; i < MT; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[q], wa[i][q], acc[i][j], 0, 0, 0);
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage has been read: the block after the next may take it
    };
    if (kb0 < kb1) {
        Block u, v;
        issue(kb0);
        load(kb0, u);
        for (int kb = kb0; kb < kb1; kb += 2) {
            if (kb + 1 < kb1) {
                issue(kb + 1);
                load(kb + 1, v);
            }
            multiply(kb, u);
            if (kb + 1 < kb1) {
                if (kb + 2 < kb1) {
                    issue(kb + 2);
                    load(kb + 2, u);
                }
                multiply(kb + 1, v);
            }
        }
    }
    // acc[i][j][e] = C[16 i + l15][n0 + 16 j + 4 h + e]
    auto part = [&](int w) { return reinterpret_cast<float*>(smem + w * 2 * STAGE); };
    const bool wide_out = g.kind == MH_F32;
    const int per = wide_out ? 4 : 8, lpr = NB * 16 / per;  // entries a thread stores, threads a row
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        if (i) __syncthreads();
#pragma unroll
        for (int j = 0; j < NB; ++j) *reinterpret_cast<f32x4*>(part(wave) + l15 * PITCH + j * 16 + h * 4) = acc[i][j];
        __syncthreads();
        for (int t = threadIdx.x; t < wn * 16 * lpr; t += 64 * RW) {
            const int gr = t / (16 * lpr), r = t / lpr % 16, c = t % lpr * per;
            const int64_t m = 16 * i + r, n = nblock + gr * (16 * NB) + c;
            if (m >= g.M || n >= g.N) continue;
            f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
            for (int w = 0; w < wk; ++w) {
                const float* p = part(gr * wk + w) + r * PITCH + c;
                lo += *reinterpret_cast<const f32x4*>(p);
                if (!wide_out) hi += *reinterpret_cast<const f32x4*>(p + 4);
            }
            float bias[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) bias[e] = g.bias && e < per && n + e < g.N ? g.bias[n + e] : 0.f;
            if (wide_out) f8_store4(g, m, n, lo[0] + bias[0], lo[1] + bias[1], lo[2] + bias[2], lo[3] + bias[3], 0);
            else f8_store8(g, m, n, lo, hi, bias, 0);
        }
    }
}

// out = sum of the slices' partial outputs, in order, + bias
__global__ __launch_bounds__(256) void fp8_join_kernel(const float* __restrict__ part, int slices, const F8Args g) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, quads = (g.N + 3) / 4;
    if (i >= g.M * quads) return;
    const int64_t m = i / quads, n = (i % quads) * 4;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    const float* p = part + m * g.N + n;
    if (g.N % 4 == 0) {
#pragma unroll 4
        for (int s = 0; s < slices; ++s) v += *reinterpret_cast<const f32x4*>(p + (int64_t)s * g.slab);
    } else {
        for (int s = 0; s < slices; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (n + e < g.N) v[e] += p[(int64_t)s * g.slab + e];
    }
    if (g.bias) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < g.N) v[e] += g.bias[n + e];
    }
    f8_store4(g, m, n, v[0], v[1], v[2], v[3], 0);
}

constexpr int64_t MOST_K = (1 << 24) - 128;  // a tile's rows lie within 32 bits of its first
constexpr int ROWS_MOST = 64;   // rows of a that the streaming kernel takes
constexpr int FUSED_MOST = 16;  // ... and quantises itself

struct F8Plan {
    bool rows, big;
    int slices, kb_split;
};
// How a product is laid out, from its sizes alone.
F8Plan f8_plan(int64_t M, int64_t N, int64_t K) {
    F8Plan p = {};
    const int kb = (int)mh_ceil_div(K, 128);
    p.slices = 1;
    p.kb_split = (kb + 3) / 4 * 4;
    // The streaming kernel's wavefronts work through the 16-row groups of a and their blocks of k one by one: too long where both are many, unless b
    // is much to read as well.  Streaming / tiles, fp32 outputs (us in a graph): 48 x 2048, 32 blocks 11.9 / 13.5, 64 blocks 19.8 / 14.6; 48 x 14341, 32
    // blocks 18.9 / 27.1, x 65536 57 / 101; 64 rows, x 2048, 16 blocks 9.9 / 14.0, 32 blocks 16.4 / 14.7; x 30000, 16 blocks 24.9 / 25.8, 32 blocks
    // 42 / 37; x 200000, 32 blocks 327 / 354 (bf16 267 / 255).
    const int64_t groups = mh_ceil_div(M, 16);
    if (M <= ROWS_MOST && (groups == 1 || groups * kb <= 96 || (groups <= 3 && N > 8192))) {
        p.rows = true;
        return p;
    }
    // Large tiles read less, and where they fill the 256 compute units' rounds they are faster: large / small, fp32 outputs, 4096 x 4096 (one full round) x
    // 128 18 / 20 us, x 4096 116 / 132; 4608 x 4096 (two rounds, 0.56 full) x 4096 180 / 151; 6144 x 4096 (0.75) x 512 42 / 40, x 4096 179 / 179 (bf16
    // 100 / 108); 7168 x 4096 (0.875) x 128 29 / 31; 8192^3 821 / 935 (bf16 417 / 513).
    const int64_t large = mh_ceil_div(M, 256) * mh_ceil_div(N, 256);
    p.big = large >= 256 && large * 100 >= mh_ceil_div(large, 256) * 256 * (kb >= 16 ? 75 : 85);
    if (!p.big) {
        // Too few tiles for the chip: slices of the summed axis, each long enough to be worth its partial output (eight blocks: 1024^3 in one slice
        // 12 us, two 16), and not more than the join reads well (128 x 415 x 65536: 64 slices 76 us, 32 51).  A tile for each of the 256 compute
        // units is enough (2048^3 bf16: 15 us, 26 in two slices); below that two workgroups a unit are better than one (1024 x 2048 x 16384: 76,
        // 116 in one slice).
        const int64_t tiles = mh_ceil_div(M, 128) * mh_ceil_div(N, 128);
        int64_t s = tiles >= 256 ? 1 : 512 / tiles;
        if (s > kb / 8) s = kb / 8;
        if (s > 32) s = 32;
        if (s > 1) {
            p.kb_split = (int)mh_ceil_div(mh_ceil_div(kb, s), 4) * 4;
            p.slices = (int)mh_ceil_div(kb, p.kb_split);
        }
    }
    return p;
}

int64_t f8_part_bytes(int64_t M, int64_t N, int64_t K) {
    const F8Plan p = f8_plan(M, N, K);
    return p.slices > 1 ? (int64_t)p.slices * M * N * 4 : 0;
}

// Launches KERN with more LDS than a launch may ask for unannounced: announced once on each device.
template <auto KERN, typename... A>
int32_t f8_launch(dim3 grid, dim3 block, int lds, hipStream_t s, A... args) {
    static std::atomic<uint64_t> announced{0};
    if (lds > 65536) {
        int dev = 0;
        (void)hipGetDevice(&dev);
        const uint64_t bit = (uint64_t)1 << (dev & 63);
        if (!(announced.load(std::memory_order_relaxed) & bit)) {
            if (hipFuncSetAttribute(reinterpret_cast<const void*>(KERN), hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) {
                (void)hipGetLastError();
                mh_set_error("mh_fp8_matmul: %d bytes of LDS refused", lds);
                return MH_ERR_LAUNCH;
            }
            announced.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    MH_LAUNCH(KERN, grid, block, lds, s, args...);
    return MH_OK;
}

template <int BM, int BN, int WM, int WN>
int32_t f8_launch_tiles(F8Args g, int slices, bool wide, hipStream_t s) {
    g.mt = (int)mh_ceil_div(g.M, BM);
    g.nt = (int)mh_ceil_div(g.N, BN);
    g.per_xcd = (int)mh_ceil_div((int64_t)g.mt * g.nt, 8);
    const dim3 grid(8 * g.per_xcd, slices), block(WM * WN * 64);
    constexpr int lds = 2 * ((BM + BN) * 128 + (BM + BN) * 4);
    return wide ? f8_launch<fp8_gemm_kernel<BM, BN, WM, WN, true>>(grid, block, lds, s, g)
                : f8_launch<fp8_gemm_kernel<BM, BN, WM, WN, false>>(grid, block, lds, s, g);
}

template <int MT, int NB, typename X>
int32_t f8_launch_rows_nb(const F8Args& g, const X* x, int64_t ldx, int K, int wk, hipStream_t s) {
    const dim3 grid((unsigned)mh_ceil_div(g.N, RW / wk * 16 * NB)), block(64 * RW);
    constexpr int lds = RW * 2 * f8_rows_stage<NB>();
    // Up to 16 rows the sums are in 32 bits for bf16 outputs as well, which costs next to nothing: reading b is the bound (8-bit instruction / widened, us: 8 x
    // 4096 -> 65536 42.8 / 43.0, 16 x 4096 -> 65536 43.2 / 43.2, 16 x 8192 -> 65536 105 / 106, 1 x 4096 -> 16384 13.1 / 13.9).  More rows: 48 x 4096 -> 14341
    // 19.3 / 21.0, 64 x 128 -> 1000000 87 / 96, 64 x 1024 -> 30000 12.9 / 15.3.
    if constexpr (MT > 1) {
        if (g.kind == MH_BF16) return f8_launch<fp8_rows_kernel<MT, NB, false, X>>(grid, block, lds, s, g, x, ldx, K, wk);
    }
    return f8_launch<fp8_rows_kernel<MT, NB, true, X>>(grid, block, lds, s, g, x, ldx, K, wk);
}
template <int MT, typename X>
int32_t f8_launch_rows(const F8Args& g, const X* x, int64_t ldx, int K, hipStream_t s) {
    // Long b: rather rows of its own for a wavefront than a short share of k, as long as there are workgroups for most of the chip and no share is longer
    // than 16 blocks (24 x 1024 -> 65536: 25 us with eight sharing, 17 with two; 48 x 2048 -> 20000: 20 in 313 workgroups, 17 in 157; 16 x 8192 -> 65536:
    // 115 with eight, 107 with four, 142 with one).
    int wk = g.kblocks >= 8 ? 8 : g.kblocks >= 4 ? 4 : g.kblocks >= 2 ? 2 : 1;
    while (wk > 1 && g.kblocks * 2 <= 16 * wk && mh_ceil_div(g.N, RW / (wk / 2) * 64) >= 150) wk /= 2;
    // As few rows of b a wavefront as still give one workgroup a compute unit: fewer leave compute units idle, and a second workgroup on some takes as long
    // as one on all (48 x 4096 -> 11000 in 344 workgroups of two groups of 16 a wavefront: 29 us, in 172 of four 19; 8192 rows in 256 of two 15.6, in
    // 128 of four 18.0; 2048 rows in 128 of one 13.0, in 64 of two 13.9).
    auto groups = [&](int nb) { return mh_ceil_div(g.N, RW / wk * 16 * nb); };
    if (groups(2) > 256) return f8_launch_rows_nb<MT, 4>(g, x, ldx, K, wk, s);
    if (groups(1) > 256) return f8_launch_rows_nb<MT, 2>(g, x, ldx, K, wk, s);
    return f8_launch_rows_nb<MT, 1>(g, x, ldx, K, wk, s);
}
int32_t f8_launch_rows_any(const F8Args& g, hipStream_t s) {
    const f8_stored* none = nullptr;
    const int mt = (int)mh_ceil_div(g.M, 16);
    if (mt == 1) return f8_launch_rows<1>(g, none, 0, 0, s);
    if (mt == 2) return f8_launch_rows<2>(g, none, 0, 0, s);
    if (mt == 3) return f8_launch_rows<3>(g, none, 0, 0, s);
    return f8_launch_rows<4>(g, none, 0, 0, s);
}

int32_t f8_check_matrix(const char* who, const char* name, const void* q, int64_t ld, const void* s, int64_t lds, int64_t rows, int64_t K) {
    const int64_t kp = mh_ceil_div(K, 128) * 128;
    MH_REQUIRE(rows == 0 || (q && s), "%s: %s is NULL", who, name);
    MH_REQUIRE(ld >= kp && ld % 16 == 0 && (reinterpret_cast<uintptr_t>(q) & 15) == 0,
               "%s: rows of %s must be 16-byte aligned and hold %lld entries (whole blocks of 128)", who, name, (long long)kp);
    MH_REQUIRE(lds >= mh_ceil_div(kp / 128, 4) * 4 && lds % 4 == 0 && lds <= 1 << 24 && (reinterpret_cast<uintptr_t>(s) & 3) == 0,
               "%s: rows of the scales of %s must be 4-byte aligned, hold a multiple of four blocks and lie at most 2^24 apart", who, name);
    return MH_OK;
}

F8Args f8_args(const uint8_t* a, int64_t lda, const uint8_t* as, int64_t ldas, const uint8_t* b, int64_t ldb, const uint8_t* bs, int64_t ldbs, int64_t M,
               int64_t N, int64_t K, const float* bias, int32_t kind, void* out, int64_t ldo) {
    F8Args g = {};
    g.a = a, g.as = as, g.b = b, g.bs = bs, g.lda = lda, g.ldas = ldas, g.ldb = ldb, g.ldbs = ldbs, g.M = M, g.N = N;
    g.kblocks = (int)mh_ceil_div(K, 128);
    g.bias = bias, g.kind = kind, g.out = out, g.ldo = ldo;
    const int64_t es = kind == MH_F32 ? 4 : 2;
    const uintptr_t at = reinterpret_cast<uintptr_t>(out);
    g.vec = ldo % 4 || at % (4 * es) ? 0 : ldo % 8 || at % (8 * es) ? 1 : 2;
    return g;
}

int32_t f8_matmul(const char* who, const uint8_t* a, int64_t lda, const uint8_t* as, int64_t ldas, const uint8_t* b, int64_t ldb, const uint8_t* bs,
                  int64_t ldbs, int64_t M, int64_t N, int64_t K, const float* bias, int32_t kind, void* out, int64_t ldo, void* ws, int64_t ws_bytes,
                  hipStream_t s) {
    F8Args g = f8_args(a, lda, as, ldas, b, ldb, bs, ldbs, M, N, K, bias, kind, out, ldo);
    const F8Plan p = f8_plan(M, N, K);
    const bool wide = kind != MH_BF16;
    g.kb_split = p.kb_split;
    if (p.rows) {
        if (int32_t rc = f8_launch_rows_any(g, s)) return rc;
        MH_CHECK_LAUNCH(who);
        return MH_OK;
    }
    F8Args t = g;
    if (p.slices > 1) {
        if (ws_bytes < f8_part_bytes(M, N, K) || !ws || (reinterpret_cast<uintptr_t>(ws) & 15)) {
            mh_set_error("%s: workspace too small or not 16-byte aligned (%lld bytes)", who, (long long)ws_bytes);
            return MH_ERR_WORKSPACE;
        }
        g.slab = t.slab = M * N;
        t.out = ws, t.ldo = N, t.kind = MH_F32, t.bias = nullptr, t.vec = N % 4 == 0;
    }
    const int32_t rc = p.big ? f8_launch_tiles<256, 256, 2, 4>(t, p.slices, wide, s) : f8_launch_tiles<128, 128, 2, 2>(t, p.slices, wide, s);
    if (rc) return rc;
    MH_CHECK_LAUNCH(who);
    if (p.slices > 1) {
        MH_LAUNCH(fp8_join_kernel, dim3((unsigned)mh_ceil_div(M * mh_ceil_div(N, 4), 256)), dim3(256), 0, s, (const float*)ws, p.slices, g);
        MH_CHECK_LAUNCH(who);
    }
    return MH_OK;
}

template <typename T>
int32_t f8_quantize_rows(const T* x, int64_t ldx, int64_t R, int64_t K, uint8_t* q, int64_t ldq, uint8_t* sc, int64_t lds, hipStream_t s) {
    const int64_t quads = mh_ceil_div(mh_ceil_div(K, 128), 4), blocks = mh_ceil_div(R, 4) * quads;
    MH_REQUIRE(blocks < (int64_t)1 << 24, "mh_fp8_quantize: matrix too large for one launch (2^32 threads)");
    MH_LAUNCH(fp8_quantize_rows_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, s, x, ldx, R, (int)K, (int)quads, q, ldq, sc, lds);
    MH_CHECK_LAUNCH("mh_fp8_quantize");
    return MH_OK;
}

// q NULL: the columns' form alone
template <typename T>
int32_t f8_quantize_tiles(const char* who, const T* x, int64_t ldx, int64_t R, int64_t C, uint8_t* q, int64_t ldq, uint8_t* sc, int64_t lds, uint8_t* qt,
                          int64_t ldqt, uint8_t* st, int64_t ldst, float* colsum, float* part, hipStream_t s) {
    const int64_t rb = mh_ceil_div(R, 128), cb = mh_ceil_div(C, 128);
    MH_REQUIRE(rb * cb < (int64_t)1 << 23 && (!colsum || mh_ceil_div(C, 64) < (int64_t)1 << 22), "%s: matrix too large for one launch (2^32 threads)", who);
    if (!colsum) part = nullptr;
    if (q) MH_LAUNCH((fp8_quantize_tiles_kernel<T, true>), dim3((unsigned)(rb * cb)), dim3(512), 0, s, x, ldx, R, C, (int)cb, (int)rb, q, ldq, sc, lds, qt, ldqt, st, ldst, part);
    else MH_LAUNCH((fp8_quantize_tiles_kernel<T, false>), dim3((unsigned)(rb * cb)), dim3(512), 0, s, x, ldx, R, C, (int)cb, (int)rb, q, ldq, sc, lds, qt, ldqt, st, ldst, part);
    MH_CHECK_LAUNCH(who);
    if (colsum) {
        MH_LAUNCH(fp8_colsum_kernel, dim3((unsigned)mh_ceil_div(C, 64)), dim3(1024), 0, s, (const float*)part, (int)rb, C, colsum);
        MH_CHECK_LAUNCH(who);
    }
    return MH_OK;
}

int32_t f8_check_source(const char* who, const void* x, int32_t dtype, int64_t ldx, int64_t R, int64_t K) {
    MH_REQUIRE(R >= 0 && K >= 0 && R < (int64_t)1 << 31 && K < (int64_t)1 << 31 && ldx >= K, "%s: sizes R=%lld K=%lld ldx=%lld", who, (long long)R,
               (long long)K, (long long)ldx);
    MH_REQUIRE(dtype == MH_F32 || dtype == MH_BF16 || dtype == MH_F16, "%s: unknown type %d", who, (int)dtype);
    MH_REQUIRE(x || R == 0 || K == 0, "%s: x is NULL", who);
    return MH_OK;
}
int32_t f8_check_sums(const char* who, const float* colsum, const void* ws, int64_t bytes, int64_t R, int64_t K) {
    if (colsum && (!ws || bytes < mh_ceil_div(R, 128) * K * 4 || (reinterpret_cast<uintptr_t>(ws) & 3))) {
        mh_set_error("%s: workspace too small or not aligned (%lld bytes)", who, (long long)bytes);
        return MH_ERR_WORKSPACE;
    }
    return MH_OK;
}

int64_t f8_q_bytes(int64_t rows, int64_t K) { return mh_ceil_div(rows * mh_ceil_div(K, 128) * 128, 256) * 256; }
int64_t f8_s_bytes(int64_t rows, int64_t K) { return mh_ceil_div(rows * mh_ceil_div(mh_ceil_div(K, 128), 4) * 4, 256) * 256; }

int32_t f8_check_out(const char* who, int64_t M, int64_t N, int64_t K, int32_t kind, const void* out, int64_t ldo) {
    MH_REQUIRE(M >= 0 && N >= 0 && K >= 1 && K <= MOST_K && M < (int64_t)1 << 27 && N < (int64_t)1 << 27, "%s: sizes M=%lld N=%lld K=%lld", who,
               (long long)M, (long long)N, (long long)K);
    MH_REQUIRE(kind == MH_F32 || kind == MH_BF16 || kind == MH_F16, "%s: unknown output type %d", who, (int)kind);
    MH_REQUIRE(ldo >= N && (out || M * N == 0), "%s: output rows of %lld entries cannot hold %lld", who, (long long)ldo, (long long)N);
    MH_REQUIRE(mh_ceil_div(M, 128) * mh_ceil_div(N, 128) < (int64_t)1 << 23, "%s: output too large for one launch (2^32 threads)", who);
    return MH_OK;
}

}  // namespace

extern "C" {

int32_t mh_fp8_quantize(const void* x, int32_t dtype, int64_t ldx, int64_t R, int64_t K, int32_t transpose, void* q, int64_t ldq, void* scales,
                        int64_t lds, float* colsum, void* workspace, int64_t workspace_bytes, mh_stream_t stream) {
    const char* const who = "mh_fp8_quantize";
    if (int32_t rc = f8_check_source(who, x, dtype, ldx, R, K)) return rc;
    MH_REQUIRE(!colsum || transpose, "mh_fp8_quantize: column sums come with transpose only");
    if (R == 0 || K == 0) return MH_OK;
    if (int32_t rc = f8_check_matrix(who, "q", q, ldq, scales, lds, transpose ? K : R, transpose ? R : K)) return rc;
    if (int32_t rc = f8_check_sums(who, colsum, workspace, workspace_bytes, R, K)) return rc;
    hipStream_t s = mh_stream(stream);
    uint8_t *qq = static_cast<uint8_t*>(q), *ss = static_cast<uint8_t*>(scales);
    auto run = [&](auto* p) {
        return transpose ? f8_quantize_tiles(who, p, ldx, R, K, nullptr, 0, nullptr, 0, qq, ldq, ss, lds, colsum, static_cast<float*>(workspace), s)
                         : f8_quantize_rows(p, ldx, R, K, qq, ldq, ss, lds, s);
    };
    if (dtype == MH_F32) return run(static_cast<const float*>(x));
    if (dtype == MH_BF16) return run(static_cast<const lp_bf16*>(x));
    return run(static_cast<const lp_f16*>(x));
}

int32_t mh_fp8_quantize_both(const void* x, int32_t dtype, int64_t ldx, int64_t R, int64_t K, void* q, int64_t ldq, void* scales, int64_t lds, void* qt,
                             int64_t ldqt, void* scales_t, int64_t ldst, float* colsum, void* workspace, int64_t workspace_bytes, mh_stream_t stream) {
    const char* const who = "mh_fp8_quantize_both";
    if (int32_t rc = f8_check_source(who, x, dtype, ldx, R, K)) return rc;
    if (R == 0 || K == 0) return MH_OK;
    if (int32_t rc = f8_check_matrix(who, "q", q, ldq, scales, lds, R, K)) return rc;
    if (int32_t rc = f8_check_matrix(who, "qt", qt, ldqt, scales_t, ldst, K, R)) return rc;
    if (int32_t rc = f8_check_sums(who, colsum, workspace, workspace_bytes, R, K)) return rc;
    hipStream_t s = mh_stream(stream);
    auto run = [&](auto* p) {
        return f8_quantize_tiles(who, p, ldx, R, K, static_cast<uint8_t*>(q), ldq, static_cast<uint8_t*>(scales), lds, static_cast<uint8_t*>(qt), ldqt,
                                 static_cast<uint8_t*>(scales_t), ldst, colsum, static_cast<float*>(workspace), s);
    };
    if (dtype == MH_F32) return run(static_cast<const float*>(x));
    if (dtype == MH_BF16) return run(static_cast<const lp_bf16*>(x));
    return run(static_cast<const lp_f16*>(x));
}

int64_t mh_fp8_matmul_workspace_bytes(int64_t M, int64_t N, int64_t K) { return M > 0 && N > 0 && K > 0 ? f8_part_bytes(M, N, K) : 0; }

int32_t mh_fp8_matmul(const void* a, int64_t lda, const void* a_scales, int64_t ldas, const void* b, int64_t ldb, const void* b_scales, int64_t ldbs,
                      int64_t M, int64_t N, int64_t K, const float* bias, int32_t out_dtype, void* out, int64_t ldo, void* workspace,
                      int64_t workspace_bytes, mh_stream_t stream) {
    if (int32_t rc = f8_check_out("mh_fp8_matmul", M, N, K, out_dtype, out, ldo)) return rc;
    if (M == 0 || N == 0) return MH_OK;
    if (int32_t rc = f8_check_matrix("mh_fp8_matmul", "a", a, lda, a_scales, ldas, M, K)) return rc;
    if (int32_t rc = f8_check_matrix("mh_fp8_matmul", "b", b, ldb, b_scales, ldbs, N, K)) return rc;
    MH_REQUIRE(lda <= 1 << 24 && ldb <= 1 << 24, "mh_fp8_matmul: rows of %lld and %lld entries (at most 2^24)", (long long)lda, (long long)ldb);
    return f8_matmul("mh_fp8_matmul", static_cast<const uint8_t*>(a), lda, static_cast<const uint8_t*>(a_scales), ldas, static_cast<const uint8_t*>(b), ldb,
                     static_cast<const uint8_t*>(b_scales), ldbs, M, N, K, bias, out_dtype, out, ldo, workspace, workspace_bytes, mh_stream(stream));
}

int64_t mh_fp8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    return M > FUSED_MOST && N > 0 && K > 0 ? f8_q_bytes(M, K) + f8_s_bytes(M, K) + f8_part_bytes(M, N, K) : 0;
}

int32_t mh_fp8_linear(const void* x, int32_t x_dtype, int64_t ldx, const void* w, int64_t ldw, const void* w_scales, int64_t ldws, int64_t M, int64_t N,
                      int64_t K, const float* bias, int32_t out_dtype, void* out, int64_t ldo, void* workspace, int64_t workspace_bytes,
                      mh_stream_t stream) {
    if (int32_t rc = f8_check_out("mh_fp8_linear", M, N, K, out_dtype, out, ldo)) return rc;
    if (M == 0 || N == 0) return MH_OK;
    if (int32_t rc = f8_check_matrix("mh_fp8_linear", "w", w, ldw, w_scales, ldws, N, K)) return rc;
    MH_REQUIRE(ldw <= 1 << 24, "mh_fp8_linear: rows of %lld entries (at most 2^24)", (long long)ldw);
    if (M <= FUSED_MOST) {
        MH_REQUIRE(x && ldx >= K, "mh_fp8_linear: x is NULL or its rows are shorter than %lld", (long long)K);
        MH_REQUIRE(x_dtype == MH_F32 || x_dtype == MH_BF16 || x_dtype == MH_F16, "mh_fp8_linear: unknown type %d", (int)x_dtype);
        const int64_t xs = x_dtype == MH_F32 ? 4 : 2, os = out_dtype == MH_F32 ? 4 : 2;
        MH_REQUIRE(!lp_shared(x, ldx * xs, K * xs, M, out, ldo * os, N * os, M), "mh_fp8_linear: out overlaps x, which up to %d rows read while out is written",
                   FUSED_MOST);
        const F8Args g = f8_args(nullptr, 0, nullptr, 0, static_cast<const uint8_t*>(w), ldw, static_cast<const uint8_t*>(w_scales), ldws, M, N, K, bias, out_dtype,
                                 out, ldo);
        hipStream_t s = mh_stream(stream);
        const int32_t rc = x_dtype == MH_F32    ? f8_launch_rows<1>(g, static_cast<const float*>(x), ldx, (int)K, s)
                           : x_dtype == MH_BF16 ? f8_launch_rows<1>(g, static_cast<const lp_bf16*>(x), ldx, (int)K, s)
                                                : f8_launch_rows<1>(g, static_cast<const lp_f16*>(x), ldx, (int)K, s);
        if (rc) return rc;
        MH_CHECK_LAUNCH("mh_fp8_linear");
        return MH_OK;
    }
    if (!workspace || workspace_bytes < mh_fp8_linear_workspace_bytes(M, N, K) || (reinterpret_cast<uintptr_t>(workspace) & 15)) {
        mh_set_error("mh_fp8_linear: workspace too small or not 16-byte aligned (%lld bytes)", (long long)workspace_bytes);
        return MH_ERR_WORKSPACE;
    }
    uint8_t* q = static_cast<uint8_t*>(workspace);
    uint8_t* sc = q + f8_q_bytes(M, K);
    uint8_t* part = sc + f8_s_bytes(M, K);
    const int64_t ldq = mh_ceil_div(K, 128) * 128, lds = mh_ceil_div(ldq / 128, 4) * 4;
    if (int32_t rc = mh_fp8_quantize(x, x_dtype, ldx, M, K, 0, q, ldq, sc, lds, nullptr, nullptr, 0, stream)) return rc;
    return f8_matmul("mh_fp8_linear", q, ldq, sc, lds, static_cast<const uint8_t*>(w), ldw, static_cast<const uint8_t*>(w_scales), ldws, M, N, K, bias,
                     out_dtype, out, ldo, part, workspace_bytes - (part - q), mh_stream(stream));
}

}  // extern "C"
