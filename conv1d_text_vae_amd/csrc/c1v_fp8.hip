// Products of 8-bit operands with a scale for each block of 128, and the quantiser that makes such operands.
//
// An operand [rows][kp] (kp = roundup(K, 128)) holds e4m3 values q; block b of 128 columns of row r has the scale byte
// s[b][r] and stands for q * 2^(s - 127).  The scales are powers of two ON PURPOSE: e4m3 is a floating-point format, so a
// power of two costs none of its relative precision (only up to one of its 18 binades of range) and scaling is exact in both
// directions.  Scales lie block-major ([block][rows rounded up to 16], 127 behind the last row): one K step of a tile reads
// them as one contiguous run.
//
// Sums are fp32.  The 8-bit matrix instructions do not give them: they add each group of eight products in a window of 13 bits
// below the group's largest one (measured: of 1 + 2^-13 the small part stays, of 1 + 2^-14 it is lost), so that outputs whose
// large products cancel lose what is left.  The values are therefore widened to bf16 with their scale applied
// (v_cvt_scalef32_pk_bf16_fp8, exact: e4m3 has four significant bits) and multiplied by v_mfma_f32_*_bf16, whose products are
// exact and whose sums are fp32 throughout, at half the 8-bit rate; one rounding to the output's type comes at the end.
#include <type_traits>
#include "c1v_common.h"

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x2_t __attribute__((ext_vector_type(2)));

constexpr int FB = C1V_FP8_BLOCK;                 // 128
__host__ __device__ static inline int64_t up16(int64_t n) { return (n + 15) & ~(int64_t)15; }

// ------------------------------------------------------------------------------------------------------
// quantiser
// ------------------------------------------------------------------------------------------------------
// Rows need not be aligned to more than their element (a slice of a wider buffer): the hardware takes 16-byte loads at any
// element boundary, the packed types tell the compiler so.
typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4_u __attribute__((ext_vector_type(4), aligned(2)));

// 8 consecutive columns of a row as fp32; columns at or past `left` give 0
__device__ __forceinline__ void load8(const float* p, int left, float* v) {
    if (left >= 8) {
        const f32x4_u a = *(const f32x4_u*)p, b = *(const f32x4_u*)(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? p[i] : 0.f;
    }
}
__device__ __forceinline__ void load8(const bf16_raw* p, int left, float* v) {
    if (left >= 8) {
        const u32x4_u a = *(const u32x4_u*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(a[i] << 16); v[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u); }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? bf16_to_f32(p[i]) : 0.f;
    }
}

// magnitude bits of a finite value; a value that is none becomes NaN (e4m3 has no infinity) and counts as 0
__device__ __forceinline__ uint32_t finite_bits(float& x) {
    const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
    const bool bad = u >= 0x7f800000u;
    x = bad ? __uint_as_float(0x7fc00000u) : x;
    return bad ? 0u : u;
}
// scale byte of a block whose largest magnitude has the bits `amax`: the smallest power of two 2^(s-127), s >= 16, with
// amax <= 448 * 2^(s-127); 448 = 1.75 * 2^8, so s = exponent - 8, one more where the mantissa is over 1.75.  127 for zeros.
// (s >= 16: the smallest e4m3 number, 2^-9, then stands for 2^-120, so that every held value is a normal bf16 number.)
__device__ __forceinline__ int scale_byte(uint32_t amax) {
    const int s = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
    return amax == 0 ? 127 : (s < 16 ? 16 : s);
}
__device__ __forceinline__ float scale_value(int s) { return __uint_as_float((uint32_t)s << 23); }               // 2^(s - 127)
// Four values -> four e4m3 bytes, divided by the scale on the way (v_cvt_scalef32_pk_fp8_*): rounded once, to nearest even (off by
// at most half a step, 2^-4 of the value); nothing saturates, the scale keeps every magnitude at 448 or less.
typedef short s16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t cvt4(float a, float b, float c, float d, float scale) {
    s16x2_t w = {0, 0};
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, a, b, scale, false);
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, c, d, scale, true));
}
__device__ __forceinline__ uint32_t cvt4(uint32_t ab, uint32_t cd, float scale) {                                  // packed bf16
    s16x2_t w = {0, 0};
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2_t, ab), scale, false);
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2_t, cd), scale, true));
}
__device__ __forceinline__ uint32_t pk_max(uint32_t a, uint32_t b) {                                                // of two halves
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, a), __builtin_bit_cast(u16x2_t, b)));
}
__device__ __forceinline__ uint32_t dpp_max(uint32_t v, uint32_t o) { return v > o ? v : o; }
// maximum over the 16 lanes of a DPP row, in all of them
__device__ __forceinline__ uint32_t max16(uint32_t v) {
    v = dpp_max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));    // quad_perm [1,0,3,2]
    v = dpp_max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));    // quad_perm [2,3,0,1]
    v = dpp_max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true));   // row_half_mirror
    v = dpp_max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xF, 0xF, true));   // row_mirror
    return v;
}

struct QuantDev {
    const void* x; int64_t rows, cols, ld;
    uint8_t* q; uint8_t* s; int64_t kp, sp;        // along the rows: [rows][kp], [kp/128][sp]
    uint8_t* qt; uint8_t* st; int64_t rp, tp;      // along the columns: [cols][rp], [rp/128][tp]
    float* colsum;                                 // [row tiles][cols] or NULL
};

// N values of a row in registers, and what quantising a run of them takes; bf16 values stay packed (half the registers, and the
// packed maxima and conversions do two at a time).
template <typename T, int N> struct Run;
template <int N> struct Run<float, N> {
    float v[N];
    __device__ __forceinline__ void load(const float* p, int left) {          // values at or past `left` are 0
#pragma unroll
        for (int i = 0; i < N; i += 8) load8(p + i, left - i > 8 ? 8 : left - i, v + i);
    }
    __device__ __forceinline__ uint32_t top() const {                         // magnitude bits of the largest value
        uint32_t u = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) u = dpp_max(u, __float_as_uint(v[i]) & 0x7fffffffu);
        return u;
    }
    __device__ __forceinline__ uint32_t finite_top() {                        // ... of the finite ones; the others become NaN
        uint32_t u = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) u = dpp_max(u, finite_bits(v[i]));
        return u;
    }
    __device__ __forceinline__ uint32_t quad(int i, float scale) const { return cvt4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], scale); }
};
template <int N> struct Run<bf16_raw, N> {
    uint32_t r[N / 2];
    __device__ __forceinline__ void load(const bf16_raw* p, int left) {
#pragma unroll
        for (int i = 0; i < N; i += 8) {
            if (left - i >= 8) {
                const u32x4_u a = *(const u32x4_u*)(p + i);
#pragma unroll
                for (int k = 0; k < 4; ++k) r[i / 2 + k] = a[k];
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    r[i / 2 + k] = (i + 2 * k < left ? (uint32_t)p[i + 2 * k] : 0u) | (i + 2 * k + 1 < left ? (uint32_t)p[i + 2 * k + 1] << 16 : 0u);
            }
        }
    }
    __device__ __forceinline__ uint32_t top() const {
        uint32_t u = 0;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) u = pk_max(u, r[i] & 0x7fff7fffu);
        return dpp_max(u << 16, u & 0xffff0000u);
    }
    __device__ __forceinline__ uint32_t finite_top() {
        uint32_t u = 0;
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            float lo = __uint_as_float(r[i] << 16), hi = __uint_as_float(r[i] & 0xffff0000u);
            u = dpp_max(u, dpp_max(finite_bits(lo), finite_bits(hi)));
            r[i] = (__float_as_uint(lo) >> 16) | (__float_as_uint(hi) & 0xffff0000u);
        }
        return u;
    }
    __device__ __forceinline__ uint32_t quad(int i, float scale) const { return cvt4(r[2 * i], r[2 * i + 1], scale); }
};

// blocks along the row: 16 lanes per block, 16 rows of one block column per workgroup (their scale bytes are one 16-byte run).
// Bound by memory when large, by one trip to it when small (1024 x 302 f32: 2.5 us)
template <typename T>
__global__ __launch_bounds__(256) void quant_rows_kernel(QuantDev d) {
    const int l = threadIdx.x & 15;
    const int64_t r = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4), kb = blockIdx.y;
    const int64_t c = kb * FB + l * 8;
    const bool in = r < d.rows;
    Run<T, 8> v;
    const int64_t left = in ? d.cols - c : 0;
    v.load((const T*)d.x + r * d.ld + c, left > 8 ? 8 : (int)left);
    uint32_t u = max16(v.top());
    if (__any(u >= 0x7f800000u)) u = max16(v.finite_top());
    const int s = scale_byte(u);
    if (l == 0) d.s[kb * d.sp + r] = (uint8_t)(in ? s : 127);
    if (!in) return;
    const float f = scale_value(s);
    *(uint2*)(d.q + r * d.kp + c) = make_uint2(v.quad(0, f), v.quad(1, f));
}

// blocks along the column (and, q given, along the row too) from ONE read of x: a 128 x 128 tile per workgroup, 8 x 8 values
// per thread in registers.  The maxima (and sums) down the columns meet in LDS, where one thread per column finishes them; the
// transposed bytes are turned in LDS and leave as whole 128-byte rows.  Up to two matrices share a launch (QuantPair).
// Bound by memory: 16384 x 2048 bf16 both ways, 135 MB, 28.5 us = 4.7 TB/s of the 5.1 that a copy reaches; two launches, one
// for each way, would read x twice.
constexpr int QT_PITCH = 136;                      // bytes per column in LDS: 8-byte aligned, columns 8 apart on other banks
// 8 x 8 values of a thread: maxima along its rows and columns, and four values down a column in 8 bits
template <typename T> struct Square;
template <> struct Square<float> {
    Run<float, 8> row[8];
    __device__ __forceinline__ float get(int i, int j) const { return row[i].v[j]; }
    __device__ __forceinline__ void maxima(uint32_t* rm, uint32_t* cm) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            rm[i] = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t u = __float_as_uint(row[i].v[j]) & 0x7fffffffu;
                rm[i] = dpp_max(rm[i], u);
                cm[j] = i ? dpp_max(cm[j], u) : u;
            }
        }
    }
    __device__ __forceinline__ uint32_t down(int i, int j, float scale) const {
        return cvt4(row[i].v[j], row[i + 1].v[j], row[i + 2].v[j], row[i + 3].v[j], scale);
    }
};
template <> struct Square<bf16_raw> {
    Run<bf16_raw, 8> row[8];
    __device__ __forceinline__ float get(int i, int j) const { return __uint_as_float(j & 1 ? row[i].r[j >> 1] & 0xffff0000u : row[i].r[j >> 1] << 16); }
    __device__ __forceinline__ void maxima(uint32_t* rm, uint32_t* cm) {
        uint32_t c2[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint32_t r2 = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t u = row[i].r[k] & 0x7fff7fffu;
                r2 = pk_max(r2, u);
                c2[k] = pk_max(c2[k], u);
            }
            rm[i] = dpp_max(r2 << 16, r2 & 0xffff0000u);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) { cm[2 * k] = c2[k] << 16; cm[2 * k + 1] = c2[k] & 0xffff0000u; }
    }
    __device__ __forceinline__ uint32_t down(int i, int j, float scale) const {
        const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;              // the same half of two rows
        const int k = j >> 1;
        return cvt4(__builtin_amdgcn_perm(row[i + 1].r[k], row[i].r[k], sel), __builtin_amdgcn_perm(row[i + 3].r[k], row[i + 2].r[k], sel), scale);
    }
};

template <typename T>
__device__ __forceinline__ void quant_tile_body(const QuantDev& d, const int64_t rt, const int64_t kb, uint8_t* lds) {
    uint32_t (*cmax)[FB] = (uint32_t (*)[FB])lds;                  // [16][128], later the transposed tile
    float (*csum)[FB] = (float (*)[FB])(lds + FB * QT_PITCH);      // [16][128]
    float* cscale = (float*)(lds + FB * QT_PITCH + 16 * FB * 4);   // [128]
    const int tid = threadIdx.x, l = tid & 15, g = tid >> 4;
    const int64_t r0 = rt * FB + g * 8, c0 = kb * FB + l * 8;
    const int rows = d.rows - r0 < 8 ? (int)(d.rows - r0) : 8, cols = d.cols - c0 < 8 ? (int)(d.cols - c0) : 8;   // may be negative
    Square<T> v;
    const T* px = (const T*)d.x + r0 * d.ld + c0;
#pragma unroll
    for (int i = 0; i < 8; ++i) { v.row[i].load(px, i < rows ? cols : 0); px += d.ld; }
    if (d.colsum) {                                                // before values that are no numbers are replaced
        float t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            t[j] = ((v.get(0, j) + v.get(1, j)) + (v.get(2, j) + v.get(3, j))) + ((v.get(4, j) + v.get(5, j)) + (v.get(6, j) + v.get(7, j)));
        *(f32x4_t*)&csum[g][l * 8] = f32x4_t{t[0], t[1], t[2], t[3]};
        *(f32x4_t*)&csum[g][l * 8 + 4] = f32x4_t{t[4], t[5], t[6], t[7]};
    }
    uint32_t rm[8], cm[8];
    v.maxima(rm, cm);
    uint32_t all = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) all = dpp_max(all, rm[i]);
    if (__any(all >= 0x7f800000u)) {                               // rare: values that are not finite become NaN and count as 0
#pragma unroll
        for (int j = 0; j < 8; ++j) cm[j] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            rm[i] = v.row[i].finite_top();
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float x = v.get(i, j);
                cm[j] = dpp_max(cm[j], finite_bits(x));
            }
        }
    }
    *(uint4*)&cmax[g][l * 8] = make_uint4(cm[0], cm[1], cm[2], cm[3]);
    *(uint4*)&cmax[g][l * 8 + 4] = make_uint4(cm[4], cm[5], cm[6], cm[7]);
    __syncthreads();
    if (tid < FB) {
        uint32_t u = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) u = dpp_max(u, cmax[i][tid]);
        const int s = scale_byte(u);
        cscale[tid] = scale_value(s);
        const int64_t c = kb * FB + tid;
        if (c < d.tp) d.st[rt * d.tp + c] = (uint8_t)(c < d.cols ? s : 127);
    } else if (d.colsum && kb * FB + tid - FB < d.cols) {
        const int c = tid - FB;
        float a = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) a += csum[i][c];
        d.colsum[rt * d.cols + kb * FB + c] = a;
    }
    if (d.q) {
        int mine = 127;
        uint8_t* pq = d.q + r0 * d.kp + c0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int s = scale_byte(max16(rm[i]));
            const float f = scale_value(s);
            if (l == i && i < rows) mine = s;
            if (i < rows) *(uint2*)pq = make_uint2(v.row[i].quad(0, f), v.row[i].quad(1, f));
            pq += d.kp;
        }
        if (l < 8 && r0 + l < d.sp) d.s[kb * d.sp + r0 + l] = (uint8_t)mine;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int c = l * 8 + j;
        const float f = cscale[c];
        *(uint2*)(lds + c * QT_PITCH + g * 8) = make_uint2(v.down(0, j, f), v.down(4, j, f));
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < 4; ++p) {                                  // 8 lanes per 128-byte row of the transposed operand
        const int c = p * 32 + (tid >> 3), o = (tid & 7) * 16;
        if (kb * FB + c < d.cols) {
            const uint2 a = *(const uint2*)(lds + c * QT_PITCH + o), b = *(const uint2*)(lds + c * QT_PITCH + o + 8);
            *(uint4*)(d.qt + (kb * FB + c) * d.rp + rt * FB + o) = make_uint4(a.x, a.y, b.x, b.y);
        }
    }
}
struct QuantPair { QuantDev d[2]; int blocks0; };
template <typename T0, typename T1>
__global__ __launch_bounds__(256, 3) void quant_tile_kernel(QuantPair p) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[FB * QT_PITCH + 16 * FB * 4 + FB * 4];
    if ((int)blockIdx.x < p.blocks0) {
        const int64_t b = blockIdx.x, tiles = p.d[0].kp / FB, rt = b / tiles;      // neighbours read neighbouring columns
        quant_tile_body<T0>(p.d[0], rt, b - rt * tiles, lds);
    } else {
        const int64_t b = (int)blockIdx.x - p.blocks0, tiles = p.d[1].kp / FB, rt = b / tiles;
        quant_tile_body<T1>(p.d[1], rt, b - rt * tiles, lds);
    }
}

// column sums from the row tiles' partial sums: sixteen runs of every sixteenth tile, added in order, whatever the number NW of
// waves that share them (a thread's loads do not wait for each other: four at a time in flight)
template <int NW>
__device__ __forceinline__ void colsum_body(const float* __restrict__ part, int64_t tiles, int64_t cols, float* __restrict__ out, int64_t block, float* red) {
    const int c64 = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t c = block * 64 + c64;
#pragma unroll
    for (int g = w; g < 16; g += NW) {
        float a = 0.f;
        if (c < cols) {
#pragma unroll 4
            for (int64_t t = g; t < tiles; t += 16) a += part[t * cols + c];
        }
        red[g * 64 + c64] = a;
    }
    __syncthreads();
    if (w == 0 && c < cols) {
        float a = red[c64];
#pragma unroll
        for (int i = 1; i < 16; ++i) a += red[i * 64 + c64];
        out[c] = a;
    }
}
__global__ __launch_bounds__(1024) void quant_colsum_kernel(const float* __restrict__ part, int64_t tiles, int64_t cols, float* __restrict__ out) {
    __shared__ float red[16 * 64];
    colsum_body<16>(part, tiles, cols, out, blockIdx.x, red);
}

static int quant_check(const c1v_fp8_quant_args* a, QuantDev& d) {
    C1V_REQUIRE(a && a->x, "fp8_quantize: null argument");
    C1V_REQUIRE(a->dtype == C1V_F32 || a->dtype == C1V_BF16, "fp8_quantize: bad dtype %d", a->dtype);
    C1V_REQUIRE(a->rows > 0 && a->cols > 0 && a->ld >= a->cols, "fp8_quantize: bad shape rows=%lld cols=%lld ld=%lld", (long long)a->rows, (long long)a->cols, (long long)a->ld);
    C1V_REQUIRE((a->q != nullptr) == (a->s != nullptr) && (a->qt != nullptr) == (a->st != nullptr) && (a->q || a->qt), "fp8_quantize: values and scales go together, one pair at least");
    C1V_REQUIRE(((uintptr_t)a->q | (uintptr_t)a->s | (uintptr_t)a->qt | (uintptr_t)a->st) % 16 == 0, "fp8_quantize: outputs must be 16-byte aligned");
    C1V_REQUIRE(!a->colsum || (a->qt && a->colsum_part), "fp8_quantize: colsum needs qt and colsum_part");
    C1V_REQUIRE(a->rows <= (1ll << 28) - 16 && a->cols <= (1ll << 22), "fp8_quantize: too large");       // 16 rows, 256 threads: below 2^32 of them
    d = QuantDev{};
    d.x = a->x; d.rows = a->rows; d.cols = a->cols; d.ld = a->ld;
    d.q = (uint8_t*)a->q; d.s = (uint8_t*)a->s; d.kp = c1v_cdiv(a->cols, FB) * FB; d.sp = up16(a->rows);
    d.qt = (uint8_t*)a->qt; d.st = (uint8_t*)a->st; d.rp = c1v_cdiv(a->rows, FB) * FB; d.tp = up16(a->cols);
    d.colsum = a->colsum ? a->colsum_part : nullptr;
    const int64_t blocks = (d.rp / FB) * (d.kp / FB);
    C1V_REQUIRE(blocks < (1ll << 24), "fp8_quantize: too large");                        // 2^32 threads in a launch
    return 0;
}
// one or two matrices with column blocks in one launch
// (finish = false: the column sums are left as partial sums, for a launch that follows)
static int quant_tiles(const c1v_fp8_quant_args* a, const c1v_fp8_quant_args* b, hipStream_t st, bool finish = true) {
    QuantPair p{};
    if (quant_check(a, p.d[0]) || (b && quant_check(b, p.d[1]))) return -1;
    p.blocks0 = (int)((p.d[0].rp / FB) * (p.d[0].kp / FB));
    const int64_t blocks = p.blocks0 + (b ? (p.d[1].rp / FB) * (p.d[1].kp / FB) : 0);
    const bool h0 = a->dtype == C1V_BF16, h1 = b ? b->dtype == C1V_BF16 : h0;
    if (h0 && h1) hipLaunchKernelGGL((quant_tile_kernel<bf16_raw, bf16_raw>), dim3((unsigned)blocks), dim3(256), 0, st, p);
    else if (h0) hipLaunchKernelGGL((quant_tile_kernel<bf16_raw, float>), dim3((unsigned)blocks), dim3(256), 0, st, p);
    else if (h1) hipLaunchKernelGGL((quant_tile_kernel<float, bf16_raw>), dim3((unsigned)blocks), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((quant_tile_kernel<float, float>), dim3((unsigned)blocks), dim3(256), 0, st, p);
    C1V_LAUNCH_CHECK();
    for (int i = 0; i < 2; ++i) {
        const c1v_fp8_quant_args* q = i ? b : a;
        if (finish && q && q->colsum) {
            hipLaunchKernelGGL(quant_colsum_kernel, dim3((unsigned)c1v_cdiv(q->cols, 64)), dim3(1024), 0, st, q->colsum_part, p.d[i].rp / FB, q->cols, q->colsum);
            C1V_LAUNCH_CHECK();
        }
    }
    return 0;
}
extern "C" int c1v_fp8_quantize(const c1v_fp8_quant_args* a, void* stream) {
    QuantDev d;
    if (quant_check(a, d)) return -1;
    hipStream_t st = (hipStream_t)stream;
    if (a->qt) return quant_tiles(a, nullptr, st);
    const dim3 grid((unsigned)c1v_cdiv(a->rows, 16), (unsigned)(d.kp / FB));
    if (a->dtype == C1V_F32) hipLaunchKernelGGL(quant_rows_kernel<float>, grid, dim3(256), 0, st, d);
    else hipLaunchKernelGGL(quant_rows_kernel<bf16_raw>, grid, dim3(256), 0, st, d);
    C1V_LAUNCH_CHECK();
    return 0;
}

// ------------------------------------------------------------------------------------------------------
// product: out[m][n] = sum_b 2^(sa[b][m] + sb[b][n] - 254) sum_{k in block b} a[m][k] b[n][k]   (+ bias[n], relu)
// ------------------------------------------------------------------------------------------------------
struct Fp8GemmDev {
    const uint8_t* a; const uint8_t* sa; int64_t sap;
    const uint8_t* b; const uint8_t* sb; int64_t sbp;
    int m, n; uint32_t kp; int nk;
    const float* bias; int relu; void* out; int64_t ldo; int out_dtype; int vec16;
    float* part; int64_t part_stride; int splits;      // splits > 1: fp32 partial sums [split][m][n rounded up to 4]
    int tiles_m, tiles_n;
};

// 32 e4m3 bytes of a lane, widened to bf16 with their block's scale: four operands of v_mfma_f32_16x16x32_bf16 (which columns
// of the block an operand covers does not matter as long as both sides agree)
struct Wide { bf16x8_t v[4]; };
__device__ __forceinline__ Wide widen(const i32x8_t& q, int s) {
    const float f = scale_value(s);
    Wide w;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bf16x2_t lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[i], f, false), hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[i], f, true);
        w.v[i >> 1][(i & 1) * 4 + 0] = lo[0]; w.v[i >> 1][(i & 1) * 4 + 1] = lo[1];
        w.v[i >> 1][(i & 1) * 4 + 2] = hi[0]; w.v[i >> 1][(i & 1) * 4 + 3] = hi[1];
    }
    return w;
}
__device__ __forceinline__ f32x4_t mfma_wide(const Wide& a, const Wide& b, f32x4_t c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[i], b.v[i], c, 0, 0, 0);
    return c;
}

template <int N> __device__ __forceinline__ void wait_vm_barrier() {
    // the DMA requests of the stage about to be read have landed, this wave's own LDS reads of the stage about to be
    // overwritten are done, and after the barrier both hold for every wave
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
__device__ __forceinline__ void glds4_so(const void* sbase, uint32_t voff, uint32_t lds_addr) {      // 4 bytes a lane
    const uint32_t a = __builtin_amdgcn_readfirstlane(lds_addr);
    const uint64_t b = (uint64_t)(uintptr_t)sbase;
    const uint32_t blo = __builtin_amdgcn_readfirstlane((uint32_t)b), bhi = __builtin_amdgcn_readfirstlane((uint32_t)(b >> 32));
    const uint64_t bs = ((uint64_t)bhi << 32) | blo;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(a), "v"(voff), "s"(bs) : "memory", "m0");
}

typedef float f32x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pk_bf16(float lo, float hi) {        // one v_cvt_pk_bf16_f32
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{lo, hi}, bf16x2_t));
}
// between a wave's LDS writes and its reads of what other lanes wrote: LDS serves a wave in order, only the compiler must keep it
__device__ __forceinline__ void wave_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
typedef uint32_t u32x2_u __attribute__((ext_vector_type(2), aligned(2)));
// four outputs of a row; the stores need no alignment beyond the type's (rows of an odd length: 1999 x 1021 x 302 in two launches
// 11.8 us with single stores, 8.6 so)
__device__ __forceinline__ void store4(const Fp8GemmDev& p, int m, int n, f32x4_t v) {
    if (m >= p.m || n >= p.n) return;
    const bool whole = n + 4 <= p.n;
    if (p.bias) {
        if (whole) v += *(const f32x4_u*)(p.bias + n);
        else
#pragma unroll
            for (int i = 0; i < 3; ++i) v[i] += n + i < p.n ? p.bias[n + i] : 0.f;
    }
    if (p.relu) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];        // a NaN stays one
    }
    const int64_t at = (int64_t)m * p.ldo + n;
    if (p.out_dtype == C1V_F32) {
        float* o = (float*)p.out + at;
        if (whole) { *(f32x4_u*)o = v; return; }
#pragma unroll
        for (int i = 0; i < 3; ++i) if (n + i < p.n) o[i] = v[i];
    } else {
        bf16_raw* o = (bf16_raw*)p.out + at;
        if (whole) { *(u32x2_u*)o = u32x2_u{pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3])}; return; }
#pragma unroll
        for (int i = 0; i < 3; ++i) if (n + i < p.n) o[i] = f32_to_bf16(v[i]);
    }
}

// Workgroup -> tile: the hardware deals consecutive workgroups to the eight XCDs in turn, each with its own L2; give every
// XCD a contiguous run of tiles, walked in bands of 8 tile rows so that a round of workgroups re-reads few operand rows.
__device__ __forceinline__ void tile_of(const Fp8GemmDev& p, int bid, int& tm, int& tn) {
    const int total = p.tiles_m * p.tiles_n, per = total / 8, rem = total % 8;
    const int x = bid & 7, i = bid >> 3;
    const int t = x * per + (x < rem ? x : rem) + i;
    constexpr int BAND = 8;
    const int band = t / (BAND * p.tiles_n), first = band * BAND;
    const int h = p.tiles_m - first < BAND ? p.tiles_m - first : BAND;
    const int in = t - band * BAND * p.tiles_n;
    tm = first + in % h;
    tn = in / h;
}

// BM x BN outputs per workgroup of WM x WN waves, K in steps of one block of 128 bytes through an NS-stage LDS ring filled by
// DMA.  An operand row of a step is 128 bytes = eight 16-byte pieces; piece c of row r lies at position c ^ ((r >> 1) & 7), so
// that the 16 rows that a fragment read touches fall on different banks.  b is the MFMA's A operand: a lane then holds four
// consecutive outputs n of one row m.  For shapes with too few tiles to fill the chip with larger ones; what bounds it is the
// time of a step's trip through memory and LDS (2048 x 1024 x 384: 5.7 us, 1024 x 1024 x 1024: 6.9 us).
template <int BM, int BN, int WM, int WN, int NS>
__device__ __forceinline__ void gemm_body(const Fp8GemmDev& p, const int tile, const int split, uint8_t* lds) {
    constexpr int NW = WM * WN, FM = BM / WM / 16, FN = BN / WN / 16, J = (BM + BN) / 8 / NW, JA = BM / 8 / NW;
    constexpr int SC = (BM + BN) * 128, STAGE = SC + 512;          // scales of a step: 256 bytes for each operand
    static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && BM <= 256 && BN <= 256 && NW % 2 == 0, "a request covers rows of one operand only");
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int tm, tn;
    tile_of(p, tile, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const int per = (p.nk + p.splits - 1) / p.splits;
    const int k0 = split * per, k1 = k0 + per < p.nk ? k0 + per : p.nk, nk = k1 - k0;
    // ---- what this wave loads: J requests of 8 rows of one operand, and 256 bytes of scales
    const uint8_t* src_a = p.a + (int64_t)m0 * p.kp + (int64_t)k0 * 128;
    const uint8_t* src_b = p.b + (int64_t)n0 * p.kp + (int64_t)k0 * 128;
    uint32_t voff[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {                                  // request j covers 8 rows: of a for j < JA, of b behind it
        const int r = ((j < JA ? j : j - JA) * NW + w) * 8 + (lane >> 3), lim = (j < JA ? p.m - m0 : p.n - n0) - 1;
        const int rc = r < lim ? r : lim;                          // rows past the end re-read the last one
        voff[j] = (uint32_t)rc * p.kp + (((lane & 7) ^ ((r >> 1) & 7)) << 4);
    }
    const bool sc_a = (w & 1) == 0;
    const int64_t scp = sc_a ? p.sap : p.sbp;
    const uint8_t* ssrc = (sc_a ? p.sa : p.sb) + (int64_t)k0 * scp;
    int64_t so = (int64_t)(sc_a ? m0 : n0) + 4 * lane;
    const uint32_t soff = (uint32_t)(so < scp - 4 ? so : scp - 4);
    const uint32_t lds0 = c1v_lds_addr(lds);
    auto issue = [&](int slot, int kt) {
        const uint32_t base = lds0 + slot * STAGE;
#pragma unroll
        for (int j = 0; j < J; ++j) c1v_glds16_so((j < JA ? src_a : src_b) + (int64_t)kt * 128, voff[j], base + (j * NW + w) * 1024);
        glds4_so(ssrc + kt * scp, soff, base + SC + (sc_a ? 0 : 256));
    };
    // ---- what this wave computes
    const int wm = w / WN, wn = w % WN;
    const int fr = lane & 15, fc = (lane >> 4) * 2, fx = (fr >> 1) & 7;
    const int o0 = fr * 128 + ((fc ^ fx) << 4), o1 = fr * 128 + (((fc + 1) ^ fx) << 4);
    const int am = wm * FM * 16, bn = wn * FN * 16;
    f32x4_t acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    auto frag = [&](const uint8_t* st, int row) {
        const i32x4_t lo = *(const i32x4_t*)(st + row * 128 + o0), hi = *(const i32x4_t*)(st + row * 128 + o1);
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
#pragma unroll
    for (int s = 0; s < NS - 1; ++s)
        if (s < nk) issue(s, s);
    int slot = 0;
    for (int kt = 0; kt < nk; ++kt) {
        if (kt + NS - 1 <= nk) wait_vm_barrier<(NS - 2) * (J + 1)>();
        else wait_vm_barrier<0>();
        if (kt + NS - 1 < nk) issue(slot == 0 ? NS - 1 : slot - 1, kt + NS - 1);
        const uint8_t* st = lds + slot * STAGE;
        Wide bf[FN];
#pragma unroll
        for (int j = 0; j < FN; ++j) bf[j] = widen(frag(st, BM + bn + j * 16), st[SC + 256 + bn + j * 16 + fr]);
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const Wide af = widen(frag(st, am + i * 16), st[SC + am + i * 16 + fr]);
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = mfma_wide(bf[j], af, acc[i][j]);
        }
        slot = slot + 1 == NS ? 0 : slot + 1;
    }
    const int q4 = (lane >> 4) * 4;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const int m = m0 + am + i * 16 + fr, n = n0 + bn + j * 16 + q4;
            if (p.splits > 1) {
                if (m < p.m && n < p.n) *(f32x4_t*)(p.part + split * p.part_stride + (int64_t)m * ((p.n + 3) & ~3) + n) = acc[i][j];
            } else {
                store4(p, m, n, acc[i][j]);
            }
        }
}
template <int BM, int BN, int WM, int WN, int NS>
__global__ __launch_bounds__(64 * WM * WN, 1) void fp8_gemm_kernel(Fp8GemmDev p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    gemm_body<BM, BN, WM, WN, NS>(p, blockIdx.x, blockIdx.y, lds);
}

// The two products of a small layer's backward pass and the column sums of its bias gradient in one launch: none of the three
// fills the chip, and they do not depend on each other (2048 x 302 -> 1024: 8 + 11 + 2 us one after the other).
struct Fp8PairDev { Fp8GemmDev g[2]; int blocks0, blocks1; const float* part; int64_t tiles, cols; float* sum; };
__global__ __launch_bounds__(256, 1) void fp8_gemm_pair_kernel(Fp8PairDev p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int b = blockIdx.x;
    if (b < p.blocks0) gemm_body<64, 64, 2, 2, 4>(p.g[0], b, 0, lds);
    else if (b < p.blocks0 + p.blocks1) gemm_body<64, 64, 2, 2, 4>(p.g[1], b - p.blocks0, 0, lds);
    else colsum_body<4>(p.part, p.tiles, p.cols, p.sum, b - p.blocks0 - p.blocks1, (float*)lds);
}

// Large shapes.  Wave tiles of 32 FM x 32 FN from 32 x 32 matrix instructions (v_mfma_f32_32x32x16_bf16: half the operand
// registers read per product of the 16 x 16 form), a K step of 128 in two halves of 64: the fragments of one half are read from
// LDS, as bytes, while the others are widened and multiplied, and the barrier of a step lies between its halves, when the other
// stage of the two-stage ring has landed and this stage's last fragments are in registers -- the matrix unit has half a step of
// work queued on either side of it.  Measured, us, bf16 / fp32 out: 8192^3 791 / 815 (1.39 / 1.35 PFLOP/s, a library's bf16
// product of that size 1.35), 4096^3 104 / 109, 16384 x 4096 x 2048 218 / 235, 2048 x 4096 x 16384 231 / 234.  Bound by the bf16
// matrix rate; what the 8-bit instructions would save (8192^3 in 450 us) costs the fp32 sums.
// The outputs of a tile leave through LDS as whole 16-byte pieces of rows; the epilogue is compiled for each combination of bias and
// relu, and loads the bias once per wave (inline branches per element cost 16384 x 4096 x 2048 9 us more).
template <bool F32, int FM, int FN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 1) void fp8_gemm32_kernel(Fp8GemmDev p) {
    constexpr int BM = 32 * FM * WM, BN = 32 * FN * WN, NW = WM * WN, J = (BM + BN) / 8 / NW, JA = BM / 8 / NW;
    constexpr int SC = (BM + BN) * 128, STAGE = SC + 512;
    static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && BM <= 256 && BN <= 256 && NW % 2 == 0, "a request covers rows of one operand only");
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int tm, tn;
    tile_of(p, blockIdx.x, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN, nk = p.nk;
    const uint8_t* src_a = p.a + (int64_t)m0 * p.kp;
    const uint8_t* src_b = p.b + (int64_t)n0 * p.kp;
    uint32_t voff[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {                                  // request j covers 8 rows: of a for j < JA, of b behind it
        const int r = ((j < JA ? j : j - JA) * NW + w) * 8 + (lane >> 3), lim = (j < JA ? p.m - m0 : p.n - n0) - 1;
        const int rc = r < lim ? r : lim;                          // rows past the end re-read the last one
        voff[j] = (uint32_t)rc * p.kp + (((lane & 7) ^ ((r >> 1) & 7)) << 4);
    }
    const bool sc_a = (w & 1) == 0;
    const int64_t scp = sc_a ? p.sap : p.sbp;
    const uint8_t* ssrc = sc_a ? p.sa : p.sb;
    const int64_t so = (int64_t)(sc_a ? m0 : n0) + 4 * lane;
    const uint32_t soff = (uint32_t)(so < scp - 4 ? so : scp - 4);
    const uint32_t lds0 = c1v_lds_addr(lds);
    auto issue = [&](int slot, int kt) {
        const uint32_t base = lds0 + slot * STAGE;
#pragma unroll
        for (int j = 0; j < J; ++j) c1v_glds16_so((j < JA ? src_a : src_b) + (int64_t)kt * 128, voff[j], base + (j * NW + w) * 1024);
        glds4_so(ssrc + kt * scp, soff, base + SC + (sc_a ? 0 : 256));
    };
    const int wm = w / WN, wn = w % WN;
    const int fr = lane & 31, fc = (lane >> 5) * 2, fx = (fr >> 1) & 7;
    const int am = wm * FM * 32, bn = wn * FN * 32;
    // byte offsets of this lane's two 16-byte pieces of a fragment row, for either half of the step
    const int oh[2][2] = {{fr * 128 + ((fc ^ fx) << 4), fr * 128 + (((fc + 1) ^ fx) << 4)},
                          {fr * 128 + (((fc + 4) ^ fx) << 4), fr * 128 + (((fc + 5) ^ fx) << 4)}};
    struct Half { i32x8_t a[FM], b[FN]; };
    auto load = [&](Half& h, int slot, int which) {
        const uint8_t* st = lds + slot * STAGE;
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const uint8_t* q = st + (BM + bn + j * 32) * 128;
            h.b[j] = __builtin_shufflevector(*(const i32x4_t*)(q + oh[which][0]), *(const i32x4_t*)(q + oh[which][1]), 0, 1, 2, 3, 4, 5, 6, 7);
        }
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const uint8_t* q = st + (am + i * 32) * 128;
            h.a[i] = __builtin_shufflevector(*(const i32x4_t*)(q + oh[which][0]), *(const i32x4_t*)(q + oh[which][1]), 0, 1, 2, 3, 4, 5, 6, 7);
        }
    };
    struct Scales { int a[FM], b[FN]; };
    auto scales = [&](Scales& s, int slot) {
        const uint8_t* st = lds + slot * STAGE + SC;
#pragma unroll
        for (int i = 0; i < FM; ++i) s.a[i] = st[am + i * 32 + fr];
#pragma unroll
        for (int j = 0; j < FN; ++j) s.b[j] = st[256 + bn + j * 32 + fr];
    };
    f32x16_t acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    auto multiply = [&](const Half& h, const Scales& s) {
        Wide bw[FN];
#pragma unroll
        for (int j = 0; j < FN; ++j) bw[j] = widen(h.b[j], s.b[j]);
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const Wide aw = widen(h.a[i], s.a[i]);
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bw[j].v[q], aw.v[q], acc[i][j], 0, 0, 0);
        }
    };
    issue(0, 0);
    if (nk > 1) { issue(1, 1); wait_vm_barrier<J + 1>(); }
    else wait_vm_barrier<0>();
    Half x, y;
    Scales sx, sy;
    load(x, 0, 0);
    scales(sx, 0);
    for (int kt = 0; kt + 1 < nk; ++kt) {
        const int slot = kt & 1;
        load(y, slot, 1);
        sy = sx;
        multiply(x, sx);
        __builtin_amdgcn_sched_barrier(0);
        wait_vm_barrier<0>();
        if (kt + 2 < nk) issue(slot, kt + 2);
        load(x, slot ^ 1, 0);
        scales(sx, slot ^ 1);
        multiply(y, sy);
        __builtin_amdgcn_sched_barrier(0);
    }
    load(y, (nk - 1) & 1, 1);
    multiply(x, sx);
    multiply(y, sx);
    // ---- epilogue (F32: fp32 out, else bf16): lane -> row m = lane & 31 of a fragment, columns 8 g + 4 (lane >> 5) .. + 3 for g = 0 .. 3
    char* out = (char*)p.out;
    const int q4 = (lane >> 5) * 4;
    // every wave has its last fragments in registers, the ring is free (before the branch: at the right edge it parts the waves)
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (p.vec16 && n0 + bn + 32 * FN <= p.n) {                     // output rows start on 16-byte boundaries
        // through LDS, 32 rows of the wave at a time, so that the stores are whole runs of a row
        constexpr int PITCH = 32 * FN * 4 + 16;
        uint8_t* mine = lds + w * 32 * PITCH;
        auto store = [&](auto to_f32, auto with_bias, auto with_relu) {
            constexpr int es = decltype(to_f32)::value ? 4 : 2, lpr = 32 * FN * es / 16, rpi = 64 / lpr;      // lanes a row, rows an instruction
            f32x4_t add[FN][4];
            if constexpr (decltype(with_bias)::value)
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int g = 0; g < 4; ++g) add[j][g] = *(const f32x4_u*)(p.bias + n0 + bn + j * 32 + g * 8 + q4);
            const int rr = lane / lpr, cc = (lane % lpr) * 16;
#pragma unroll
            for (int i = 0; i < FM; ++i) {
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        f32x4_t v = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                        const int nl = j * 32 + g * 8 + q4;
                        if constexpr (decltype(with_bias)::value) v += add[j][g];
                        if constexpr (decltype(with_relu)::value)
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[e] = v[e] < 0.f ? 0.f : v[e];
                        if constexpr (decltype(to_f32)::value) *(f32x4_t*)(mine + fr * PITCH + nl * 4) = v;
                        else *(uint2*)(mine + fr * PITCH + nl * 2) = make_uint2(pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3]));
                    }
                wave_lds_sync();
#pragma unroll
                for (int r = 0; r < 32; r += rpi) {
                    const int m = m0 + am + i * 32 + r + rr;
                    const uint4 v = *(const uint4*)(mine + (r + rr) * PITCH + cc);
                    if (m < p.m) *(uint4*)(out + ((int64_t)m * p.ldo + n0 + bn) * es + cc) = v;
                }
                wave_lds_sync();
            }
        };
        const std::bool_constant<F32> f32{};
        const std::true_type yes{};
        const std::false_type no{};
        if (p.bias) { if (p.relu) store(f32, yes, yes); else store(f32, yes, no); }
        else if (p.relu) store(f32, no, yes);
        else store(f32, no, no);
        return;
    }
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4_t v = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
                const int m = m0 + am + i * 32 + fr, n = n0 + bn + j * 32 + g * 8 + q4;
                store4(p, m, n, v);
            }
}

// partial sums of the K splits, in their order
__global__ __launch_bounds__(256) void fp8_reduce_kernel(Fp8GemmDev p) {
    const int n4 = (p.n + 3) >> 2;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)p.m * n4) return;
    const float* s = p.part + i * 4;
    f32x4_t v = *(const f32x4_t*)s;
    for (int k = 1; k < p.splits; ++k) {
        const f32x4_t o = *(const f32x4_t*)(s + k * p.part_stride);
        v += o;
    }
    store4(p, (int)(i / n4), (int)(i % n4) * 4, v);
}

static int launch_tiles(const void* f, Fp8GemmDev& p, int bm, int bn, int threads, int lds, int* set, hipStream_t st) {
    p.tiles_m = (int)c1v_cdiv(p.m, bm); p.tiles_n = (int)c1v_cdiv(p.n, bn);
    int dev = 0;
    (void)hipGetDevice(&dev);
    if (*set != dev) {
        const hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        C1V_REQUIRE(e == hipSuccess, "fp8_gemm: %s", hipGetErrorString(e));
        *set = dev;
    }
    void* args[] = {&p};
    (void)hipLaunchKernel(f, dim3((unsigned)(p.tiles_m * p.tiles_n), (unsigned)p.splits), dim3((unsigned)threads), args, (size_t)lds, st);
    C1V_LAUNCH_CHECK();
    if (p.splits > 1) {
        const int64_t n = (int64_t)p.m * ((p.n + 3) >> 2);
        hipLaunchKernelGGL(fp8_reduce_kernel, dim3((unsigned)c1v_cdiv(n, 256)), dim3(256), 0, st, p);
        C1V_LAUNCH_CHECK();
    }
    return 0;
}
template <int BM, int BN, int WM, int WN, int NS>
static int launch_gemm(Fp8GemmDev& p, hipStream_t st) {
    constexpr int bytes = NS * ((BM + BN) * 128 + 512);
    static_assert(bytes <= 160 * 1024, "LDS");
    static thread_local int set = -1;
    return launch_tiles((const void*)fp8_gemm_kernel<BM, BN, WM, WN, NS>, p, BM, BN, 64 * WM * WN, bytes, &set, st);
}
template <bool F32, int FM, int FN, int WM, int WN>
static int launch_gemm32(Fp8GemmDev& p, hipStream_t st) {
    constexpr int BM = 32 * FM * WM, BN = 32 * FN * WN, ring = 2 * ((BM + BN) * 128 + 512), rows = WM * WN * 32 * (32 * FN * 4 + 16), bytes = ring > rows ? ring : rows;
    static_assert(bytes <= 160 * 1024, "LDS");
    static thread_local int set = -1;
    return launch_tiles((const void*)fp8_gemm32_kernel<F32, FM, FN, WM, WN>, p, BM, BN, 64 * WM * WN, bytes, &set, st);
}

struct Fp8Plan { int tile; int splits; };
// Which kernel, by the work there is for 256 CUs (us, bf16 out, operands in cache; tiles 64: 16 x 16 instructions, four stages;
// 128: two workgroups per CU; 256: eight waves, one workgroup per CU):
//   2048 x 1024 x 384    64: 5.7   128: 6.6   256: 12      4096 x 2048 x 640     128: 14    256: 19
//   1024 x 1024 x 1024   64: 6.9   128: 11    256: 23      4096 x 4096 x 4096    128: 120   256: 104
//   2048 x 1024 x 2048   64: 15    128: 18    256: 42      16384 x 4096 x 2048   128: 241   256: 218
//   2048 x 1300 x 640    64: 10.3  128: 10.1  256: 20      2048 x 4096 x 16384   128: 234   256: 306 (half the chip)
//   2048 x 2048 x 2048   64: 29    128: 21    256: 44      8192 x 8192 x 8192    128: 890   256: 808
// The 128 / 256 choice compares rounds of workgroups times steps (1.7 us a step with 512 slots, 3.0 us with 256) plus 6 / 8 us
// a round.  A long K of few tiles is cut into runs whose fp32 sums a second launch adds in order (us, whole / two / four):
//   256 x 512, 16 blocks 10.0 / 8.5 / 7.8    512 x 512, 16 blocks 10.1 / 9.2 / 8.7     512 x 1024, 16 blocks 10.3 / 10.6 / 12.1
//              32 blocks 17.3 / 12.1 / 9.6              32 blocks 17.5 / 12.7 / 10.6               32 blocks 17.4 / 14.3 / 15.3
//              64 blocks 32 / 19.5 / 13.3               64 blocks 32 / 20.5 / 14.5                 64 blocks 32 / 21.5 / 19.4
//   768 x 1024, 32 blocks 17.6 / 18.8 / 18.8 (192 tiles; 48 blocks 25 / 22.5 / 22.3)
// A product by itself would be ahead in runs from 16 blocks; they start at 32 because a training layer's two products share a launch
// only whole (backward of 2048 x 302 -> 128: 15.3 us together, 17.5 apart with runs; 3000 rows 19.9 / 19.2, 4096 rows 23.6 / 20.1)
// and a gradient has to have the same bits whichever others are asked for.
static Fp8Plan fp8_plan(int64_t m, int64_t n, int64_t kp) {
    const int64_t nk = kp / FB;
    const int64_t t64 = c1v_cdiv(m, 64) * c1v_cdiv(n, 64), t128 = c1v_cdiv(m, 128) * c1v_cdiv(n, 128), t256 = c1v_cdiv(m, 256) * c1v_cdiv(n, 256);
    Fp8Plan p{0, 1};
    if (t128 >= 160) {
        const double c128 = (double)c1v_cdiv(t128, 512) * (1.7 * nk + 6), c256 = (double)c1v_cdiv(t256, 256) * (3.0 * nk + 8);
        p.tile = c256 < c128 ? 2 : 1;
        return p;
    }
    if (nk >= 32 && t64 <= 128) p.splits = t64 <= 64 ? 4 : 2;
    return p;
}

extern "C" int64_t c1v_fp8_gemm_work(int64_t m, int64_t n, int64_t kp) {
    const Fp8Plan pl = fp8_plan(m, n, kp);
    return pl.splits > 1 ? (int64_t)pl.splits * m * ((n + 3) & ~(int64_t)3) * 4 : 0;
}

static int gemm_setup(const c1v_fp8_gemm_args* a, Fp8GemmDev& p, Fp8Plan& pl) {
    C1V_REQUIRE(a && a->a && a->sa && a->b && a->sb && a->out, "fp8_gemm: null argument");
    C1V_REQUIRE(a->m > 0 && a->n > 0 && a->kp > 0 && a->kp % FB == 0, "fp8_gemm: bad shape m=%lld n=%lld kp=%lld (kp: whole blocks of 128)", (long long)a->m, (long long)a->n, (long long)a->kp);
    C1V_REQUIRE(a->m < (1ll << 30) && a->n < (1ll << 30) && a->kp < (1ll << 24), "fp8_gemm: too large");
    C1V_REQUIRE(a->out_dtype == C1V_F32 || a->out_dtype == C1V_BF16, "fp8_gemm: bad out_dtype %d", a->out_dtype);
    C1V_REQUIRE(a->ldo >= a->n, "fp8_gemm: ldo (%lld) is smaller than n", (long long)a->ldo);
    C1V_REQUIRE(((uintptr_t)a->a | (uintptr_t)a->b | (uintptr_t)a->sa | (uintptr_t)a->sb) % 16 == 0, "fp8_gemm: operands must be 16-byte aligned");
    pl = fp8_plan(a->m, a->n, a->kp);
    const int64_t need = c1v_fp8_gemm_work(a->m, a->n, a->kp);
    C1V_REQUIRE(need == 0 || (a->work && a->work_bytes >= need && (uintptr_t)a->work % 16 == 0), "fp8_gemm: workspace of %lld bytes needed (c1v_fp8_gemm_work)", (long long)need);
    p = Fp8GemmDev{};
    p.a = (const uint8_t*)a->a; p.sa = (const uint8_t*)a->sa; p.sap = up16(a->m);
    p.b = (const uint8_t*)a->b; p.sb = (const uint8_t*)a->sb; p.sbp = up16(a->n);
    p.m = (int)a->m; p.n = (int)a->n; p.kp = (uint32_t)a->kp; p.nk = (int)(a->kp / FB);
    p.bias = a->bias; p.relu = a->relu; p.out = a->out; p.ldo = a->ldo; p.out_dtype = a->out_dtype;
    const int es = c1v_esize(a->out_dtype);
    p.vec16 = a->ldo * es % 16 == 0 && (uintptr_t)a->out % 16 == 0;
    p.splits = pl.splits; p.part = a->work; p.part_stride = a->m * ((a->n + 3) & ~(int64_t)3);
    return 0;
}
extern "C" int c1v_fp8_gemm(const c1v_fp8_gemm_args* a, void* stream) {
    Fp8GemmDev p;
    Fp8Plan pl;
    if (gemm_setup(a, p, pl)) return -1;
    hipStream_t st = (hipStream_t)stream;
    const bool f32 = a->out_dtype == C1V_F32;
    if (pl.tile == 2) return f32 ? launch_gemm32<true, 4, 2, 2, 4>(p, st) : launch_gemm32<false, 4, 2, 2, 4>(p, st);
    if (pl.tile == 1) return f32 ? launch_gemm32<true, 2, 2, 2, 2>(p, st) : launch_gemm32<false, 2, 2, 2, 2>(p, st);
    return launch_gemm<64, 64, 2, 2, 4>(p, st);
}

// ------------------------------------------------------------------------------------------------------
// a few rows (serving): x [rows <= 16][K] is quantised on the way into the product, one launch
// ------------------------------------------------------------------------------------------------------
struct Fp8RowsDev {
    const void* x; int64_t ldx; int rows, k;
    Fp8GemmDev p;                                  // a / sa unused
};

// Up to 16 rows the product reads n x kp weight bytes once and does 2 rows operations with each: it is bound by those bytes.
// (With more rows, fp8_dense_direct, it is a matter of latency.)  A workgroup takes 16 rows and 16 F columns; its NW waves take
// the blocks of K in turn, quantise x's block in registers exactly as the quantiser does (lane: row lane & 15, columns
// 16 (lane >> 4) .. + 15 and the same 64 further on: four lanes read whole stretches of a row, and which columns an operand's
// lane holds does not matter as long as both sides agree) and feed the weights from memory straight into the MFMA; the waves'
// sums meet in LDS in the waves' order.  Lanes of rows that x does not have repeat its last row: their products belong to
// columns of the result that nobody stores.  F fragments per block share the work of quantising x, which would otherwise cost
// more than the weights' bytes.  13 x 8192 x 4096 bf16 with the weights from memory: 11.2 us for 34 MB, of which 3.5 are what a
// launch of one block per wave takes (1 x 1024 x 1024); requesting weights two or three blocks further ahead gained nothing.
template <typename T, int F, int NW>
__global__ __launch_bounds__(64 * NW) void fp8_rows_kernel(Fp8RowsDev d) {
    __shared__ f32x4_t red[NW][F][64];
    const Fp8GemmDev& p = d.p;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int r = lane & 15, quarter = lane >> 4;
    const int n0 = blockIdx.x * (16 * F), m = blockIdx.y * 16 + r;
    const T* xr = (const T*)d.x + (int64_t)(m < d.rows ? m : d.rows - 1) * d.ldx + quarter * 16;
    const uint8_t* br[F];
    int nr[F];
#pragma unroll
    for (int f = 0; f < F; ++f) {
        nr[f] = n0 + 16 * f + r < p.n ? n0 + 16 * f + r : p.n - 1;
        br[f] = p.b + (int64_t)nr[f] * p.kp + quarter * 16;
    }
    f32x4_t acc[F];
#pragma unroll
    for (int f = 0; f < F; ++f) acc[f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    i32x4_t lo[F], hi[F], lo2[F], hi2[F];
    int bs[F], bs2[F];
    Run<T, 16> v, v2;
    auto weights = [&](int kb, i32x4_t* l, i32x4_t* h, int* s) {
#pragma unroll
        for (int f = 0; f < F; ++f) {
            l[f] = *(const i32x4_t*)(br[f] + (int64_t)kb * 128);
            h[f] = *(const i32x4_t*)(br[f] + (int64_t)kb * 128 + 64);
            s[f] = p.sb[kb * p.sbp + nr[f]];
        }
    };
    auto rows = [&](int kb) {
        const T* x = xr + (int64_t)kb * 128;
        const int left = d.k - kb * 128 - quarter * 16;
        if (kb * 128 + 128 <= d.k) { v.load(x, 16); v2.load(x + 64, 16); }
        else { v.load(x, left); v2.load(x + 64, left - 64); }
    };
    if (w < p.nk) { weights(w, lo, hi, bs); rows(w); }
    for (int kb = w; kb < p.nk; kb += NW) {
        const int next = kb + NW;
        if (next < p.nk) weights(next, lo2, hi2, bs2);             // the next block's weights are on the way meanwhile
        uint32_t u = dpp_max(v.top(), v2.top());
        u = dpp_max(u, (uint32_t)__shfl_xor((int)u, 16, 64));
        u = dpp_max(u, (uint32_t)__shfl_xor((int)u, 32, 64));
        if (__any(u >= 0x7f800000u)) {
            u = v.finite_top();
            u = dpp_max(u, v2.finite_top());
            u = dpp_max(u, (uint32_t)__shfl_xor((int)u, 16, 64));
            u = dpp_max(u, (uint32_t)__shfl_xor((int)u, 32, 64));
        }
        const int as = scale_byte(u);
        const float s = scale_value(as);
        i32x8_t af;
#pragma unroll
        for (int i = 0; i < 4; ++i) { af[i] = (int)v.quad(i, s); af[4 + i] = (int)v2.quad(i, s); }
        if (next < p.nk) rows(next);
        const Wide aw = widen(af, as);
#pragma unroll
        for (int f = 0; f < F; ++f) acc[f] = mfma_wide(widen(__builtin_shufflevector(lo[f], hi[f], 0, 1, 2, 3, 4, 5, 6, 7), bs[f]), aw, acc[f]);
#pragma unroll
        for (int f = 0; f < F; ++f) { lo[f] = lo2[f]; hi[f] = hi2[f]; bs[f] = bs2[f]; }
    }
#pragma unroll
    for (int f = 0; f < F; ++f) red[w][f][lane] = acc[f];
    __syncthreads();
    for (int f = w; f < F; f += NW) {
        f32x4_t v4 = red[0][f][lane];
#pragma unroll
        for (int i = 1; i < NW; ++i) v4 += red[i][f][lane];
        store4(p, m, n0 + 16 * f + 4 * quarter, v4);
    }
}
// Whether x is quantised inside the product's launch.  Up to 16 rows always.  Beyond, a workgroup's K is walked eight blocks at
// a time and x is quantised again for every 16 to 64 columns, against two launches and 64 x 64 tiles that walk K one block at
// a time.  Measured (us, f32 / bf16 x, back to back), here, and in two launches:
//   256 x 512 x 1920   8.1 / 6.6,    11.9 / 12.0      512 x 512 x 512    4.7 / 4.1,    6.7 / 6.8
//   256 x 1024 x 1024  6.4 / 5.4,    8.5 / 8.5        4096 x 64 x 302    4.8 / 4.7,    6.8 / 7.0
//   1024 x 1024 x 302  15.6 / 14.7,  6.9 / 7.0        512 x 1024 x 302   8.3 / 8.3,    6.6 / 6.7   (1024 and 512 workgroups)
//   256 x 512 x 2048   8.2 / 6.6,    12.3 / 12.5      256 x 512 x 2560   9.3 / 7.6,    14.4 / 14.5
//   256 x 512 x 4096   13.9 / 10.0,  12.6 / 12.4      128 x 512 x 4096   11.7 / 8.1,   11.4 / 11.4    (K in runs in two launches)
// At two turns of eight blocks no shape loses by the one launch; it would still be ahead up to 31 blocks.
static bool fp8_dense_direct(int64_t m, int64_t n, int64_t kp) {
    return m <= C1V_FP8_ROWS || (c1v_cdiv(m, 16) * c1v_cdiv(n, 64) <= 256 && kp <= 16 * FB);
}
extern "C" int c1v_fp8_dense_direct(int64_t m, int64_t n, int64_t kp) { return fp8_dense_direct(m, n, kp) ? 1 : 0; }

template <typename T, int F>
static void launch_rows1(const Fp8RowsDev& d, hipStream_t st) {
    const dim3 grid((unsigned)c1v_cdiv(d.p.n, 16 * F), (unsigned)c1v_cdiv(d.rows, 16));
    hipLaunchKernelGGL((fp8_rows_kernel<T, F, 8>), grid, dim3(512), 0, st, d);
}
// One fragment column per workgroup gives the most workgroups, two or four share the work of quantising x and its reads: the fewest
// that keep to one workgroup per CU.  Measured (us, bf16 / f32 x, weights from memory for up to 16 rows), 1 / 2 / 4:
//   13 x 4096 x 1024   4.3 4.6 5.6 / 4.8 5.3 6.3       8 x 4112 x 1024    4.5 4.4 5.3 / 5.6 4.9 5.9
//   1 x 4096 x 4096    8.3 8.8 12.6 / 9.1 10.3 14.3    1 x 4112 x 4096    10.0 8.9 12.6 / 11.9 10.4 14.3
//   1 x 8192 x 4096    12.6 10.7 13.1 / 13.8 12.2 15.0 1 x 8208 x 4096    14.7 14.4 13.2 / 17.7 18.2 15.0
//   13 x 8192 x 4096   15.2 11.5 15.0 / 19.9 14.6 17.3 13 x 12288 x 4096  21.2 18.6 15.5 / 27.1 25.2 18.4
//   64 x 512 x 1920    5.2 6.2 8.0 / 6.6 7.8 9.7       256 x 512 x 1920   8.0 6.4 8.1 / 11.2 7.9 9.7
//   17 x 4096 x 1024   4.7 4.3 5.3 / 5.7 5.2 6.2       512 x 512 x 512    5.9 4.4 4.1 / 7.6 6.3 4.7
// (sixteen waves instead of eight: no faster anywhere).
template <typename T>
static void launch_rows(const Fp8RowsDev& d, hipStream_t st) {
    const int64_t rt = c1v_cdiv(d.rows, 16);
    if (rt * c1v_cdiv(d.p.n, 16) <= 256) launch_rows1<T, 1>(d, st);
    else if (rt * c1v_cdiv(d.p.n, 32) <= 256) launch_rows1<T, 2>(d, st);
    else launch_rows1<T, 4>(d, st);
}

extern "C" int c1v_fp8_dense(const c1v_fp8_dense_args* a, void* stream) {
    C1V_REQUIRE(a && a->x && a->g.b && a->g.sb && a->g.out, "fp8_dense: null argument");
    C1V_REQUIRE(a->x_dtype == C1V_F32 || a->x_dtype == C1V_BF16, "fp8_dense: bad x_dtype %d", a->x_dtype);
    C1V_REQUIRE(a->g.m > 0 && a->k > 0 && a->ldx >= a->k && c1v_cdiv(a->k, FB) * FB == a->g.kp, "fp8_dense: bad shape rows=%lld k=%lld ldx=%lld kp=%lld",
                (long long)a->g.m, (long long)a->k, (long long)a->ldx, (long long)a->g.kp);
    if (!fp8_dense_direct(a->g.m, a->g.n, a->g.kp)) {
        c1v_fp8_quant_args q{};
        q.x = a->x; q.dtype = a->x_dtype; q.rows = a->g.m; q.cols = a->k; q.ld = a->ldx; q.q = (void*)a->g.a; q.s = (void*)a->g.sa;
        C1V_REQUIRE(q.q && q.s, "fp8_dense: %lld rows need room for the quantised rows (g.a, g.sa)", (long long)a->g.m);
        const int rc = c1v_fp8_quantize(&q, stream);
        return rc ? rc : c1v_fp8_gemm(&a->g, stream);
    }
    const c1v_fp8_gemm_args& g = a->g;
    C1V_REQUIRE(g.n > 0 && g.n < (1ll << 27) && g.m < (1ll << 20) && g.kp < (1ll << 24) && g.ldo >= g.n, "fp8_dense: bad shape n=%lld ldo=%lld", (long long)g.n, (long long)g.ldo);
    C1V_REQUIRE(g.out_dtype == C1V_F32 || g.out_dtype == C1V_BF16, "fp8_dense: bad out_dtype %d", g.out_dtype);
    C1V_REQUIRE(((uintptr_t)g.b | (uintptr_t)g.sb) % 16 == 0, "fp8_dense: weights must be 16-byte aligned");
    Fp8RowsDev d{};
    d.x = a->x; d.ldx = a->ldx; d.rows = (int)g.m; d.k = (int)a->k;
    d.p.b = (const uint8_t*)g.b; d.p.sb = (const uint8_t*)g.sb; d.p.sbp = up16(g.n);
    d.p.m = (int)g.m; d.p.n = (int)g.n; d.p.kp = (uint32_t)g.kp; d.p.nk = (int)(g.kp / FB);
    d.p.bias = g.bias; d.p.relu = g.relu; d.p.out = g.out; d.p.ldo = g.ldo; d.p.out_dtype = g.out_dtype;
    if (a->x_dtype == C1V_F32) launch_rows<float>(d, (hipStream_t)stream);
    else launch_rows<bf16_raw>(d, (hipStream_t)stream);
    C1V_LAUNCH_CHECK();
    return 0;
}

// ------------------------------------------------------------------------------------------------------
// a dense layer in training: y = x W + bias and its gradients, every product in 8 bits
// ------------------------------------------------------------------------------------------------------
// Buffers in the caller's `keep` (held from forward to backward) and `temp`, in this order, each on a 256-byte boundary.
namespace {
struct Carver {
    char* base; int64_t at;
    void* take(int64_t bytes) { void* p = base ? base + at : nullptr; at += (bytes + 255) & ~(int64_t)255; return p; }
    void operand(int64_t rows, int64_t cols, void*& q, void*& s) {      // [rows][cols] in 8 bits
        const int64_t kp = c1v_cdiv(cols, FB) * FB;
        q = take(rows * kp); s = take(kp / FB * up16(rows));
    }
};
struct LinearBufs {
    void *qx, *sx, *qkt, *skt;                     // forward operands (temp)
    void *qxt, *sxt, *qk, *sk;                     // backward operands of x and the kernel (keep)
    void *qd, *sd, *qdt, *sdt; float* part;        // backward operands of dy (temp)
    float* work; int64_t work_bytes;
    int64_t keep, temp;
};
LinearBufs linear_fwd_bufs(const c1v_fp8_linear_args* a, void* keep, void* temp) {
    LinearBufs b{};
    Carver k{(char*)keep, 0}, t{(char*)temp, 0};
    if (a->need_dx) k.operand(a->k, a->n, b.qk, b.sk);
    if (a->need_dk) k.operand(a->k, a->rows, b.qxt, b.sxt);
    t.operand(a->rows, a->k, b.qx, b.sx);
    t.operand(a->n, a->k, b.qkt, b.skt);
    b.work_bytes = c1v_fp8_gemm_work(a->rows, a->n, c1v_cdiv(a->k, FB) * FB);
    b.work = (float*)t.take(b.work_bytes);
    b.keep = k.at; b.temp = t.at;
    return b;
}
LinearBufs linear_bwd_bufs(const c1v_fp8_linear_args* a, void* keep, void* temp) {
    LinearBufs b{};
    Carver k{(char*)keep, 0}, t{(char*)temp, 0};
    if (a->need_dx) k.operand(a->k, a->n, b.qk, b.sk);
    if (a->need_dk) k.operand(a->k, a->rows, b.qxt, b.sxt);
    if (a->need_dx) t.operand(a->rows, a->n, b.qd, b.sd);
    if (a->need_dk || a->need_db) t.operand(a->n, a->rows, b.qdt, b.sdt);
    if (a->need_db) b.part = (float*)t.take(c1v_cdiv(a->rows, FB) * a->n * 4);
    const int64_t w0 = a->need_dx ? c1v_fp8_gemm_work(a->rows, a->k, c1v_cdiv(a->n, FB) * FB) : 0;
    const int64_t w1 = a->need_dk ? c1v_fp8_gemm_work(a->k, a->n, c1v_cdiv(a->rows, FB) * FB) : 0;
    b.work_bytes = w0 > w1 ? w0 : w1;
    b.work = (float*)t.take(b.work_bytes);
    b.keep = k.at; b.temp = t.at;
    return b;
}
int linear_check(const c1v_fp8_linear_args* a, const char* what) {
    C1V_REQUIRE(a, "%s: null argument", what);
    C1V_REQUIRE(a->rows > 0 && a->k > 0 && a->n > 0, "%s: bad shape rows=%lld k=%lld n=%lld", what, (long long)a->rows, (long long)a->k, (long long)a->n);
    C1V_REQUIRE(a->rows <= (1ll << 24) - FB || (!a->need_dk && a->rows <= (1ll << 28) - 16), "%s: too many rows (%lld; the kernel's gradient takes up to 2^24 - 128)", what, (long long)a->rows);
    C1V_REQUIRE(a->k <= (1ll << 22) && a->n <= (1ll << 22), "%s: too large", what);
    C1V_REQUIRE((a->x_dtype == C1V_F32 || a->x_dtype == C1V_BF16) && (a->k_dtype == C1V_F32 || a->k_dtype == C1V_BF16), "%s: bad dtype", what);
    C1V_REQUIRE(((uintptr_t)a->keep | (uintptr_t)a->temp) % 16 == 0, "%s: keep and temp must be 16-byte aligned", what);
    return 0;
}
c1v_fp8_gemm_args linear_gemm(const void* a, const void* sa, const void* b, const void* sb, int64_t m, int64_t n, int64_t k, const float* bias, int dtype,
                              void* out, const LinearBufs& w) {
    c1v_fp8_gemm_args g{};
    g.a = a; g.sa = sa; g.b = b; g.sb = sb; g.m = m; g.n = n; g.kp = c1v_cdiv(k, FB) * FB; g.bias = bias; g.out_dtype = dtype; g.out = out; g.ldo = n;
    g.work = w.work; g.work_bytes = w.work_bytes;
    return g;
}
int launch_pair(const Fp8PairDev& p, unsigned blocks, hipStream_t st) {
    constexpr int bytes = 4 * ((64 + 64) * 128 + 512);
    static thread_local int set = -1;
    int dev = 0;
    (void)hipGetDevice(&dev);
    if (set != dev) {
        const hipError_t e = hipFuncSetAttribute((const void*)fp8_gemm_pair_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
        C1V_REQUIRE(e == hipSuccess, "fp8_linear_bwd: %s", hipGetErrorString(e));
        set = dev;
    }
    hipLaunchKernelGGL(fp8_gemm_pair_kernel, dim3(blocks), dim3(256), bytes, st, p);
    C1V_LAUNCH_CHECK();
    return 0;
}
}

extern "C" int c1v_fp8_linear_sizes(const c1v_fp8_linear_args* a, int64_t* keep, int64_t* temp_fwd, int64_t* temp_bwd) {
    if (linear_check(a, "fp8_linear_sizes")) return -1;
    C1V_REQUIRE(keep && temp_fwd && temp_bwd, "fp8_linear_sizes: null argument");
    const LinearBufs f = linear_fwd_bufs(a, nullptr, nullptr), b = linear_bwd_bufs(a, nullptr, nullptr);
    *keep = f.keep; *temp_fwd = f.temp; *temp_bwd = b.temp;
    return 0;
}
extern "C" int c1v_fp8_linear_fwd(const c1v_fp8_linear_args* a, void* stream) {
    if (linear_check(a, "fp8_linear_fwd")) return -1;
    C1V_REQUIRE(a->x && a->kernel && a->y && a->temp && (a->keep || !(a->need_dx || a->need_dk)), "fp8_linear_fwd: null argument");
    const LinearBufs b = linear_fwd_bufs(a, a->keep, a->temp);
    c1v_fp8_quant_args q{}, w{};
    q.x = a->x; q.dtype = a->x_dtype; q.rows = a->rows; q.cols = a->k; q.ld = a->ldx; q.q = b.qx; q.s = b.sx; q.qt = b.qxt; q.st = b.sxt;
    w.x = a->kernel; w.dtype = a->k_dtype; w.rows = a->k; w.cols = a->n; w.ld = a->ldk; w.q = b.qk; w.s = b.sk; w.qt = b.qkt; w.st = b.skt;
    int rc = a->need_dk ? quant_tiles(&q, &w, (hipStream_t)stream) : c1v_fp8_quantize(&q, stream);
    if (!rc && !a->need_dk) rc = c1v_fp8_quantize(&w, stream);
    if (rc) return rc;
    const c1v_fp8_gemm_args g = linear_gemm(b.qx, b.sx, b.qkt, b.skt, a->rows, a->n, a->k, a->bias, a->x_dtype, a->y, b);
    return c1v_fp8_gemm(&g, stream);
}
extern "C" int c1v_fp8_linear_bwd(const c1v_fp8_linear_args* a, void* stream) {
    if (linear_check(a, "fp8_linear_bwd")) return -1;
    C1V_REQUIRE(a->dy && a->temp && (a->keep || !(a->need_dx || a->need_dk)), "fp8_linear_bwd: null argument");
    C1V_REQUIRE((a->dx || !a->need_dx) && (a->dk || !a->need_dk) && (a->db || !a->need_db), "fp8_linear_bwd: null gradient");
    if (!a->need_dx && !a->need_dk && !a->need_db) return 0;
    const LinearBufs b = linear_bwd_bufs(a, a->keep, a->temp);
    c1v_fp8_quant_args q{};
    q.x = a->dy; q.dtype = a->x_dtype; q.rows = a->rows; q.cols = a->n; q.ld = a->ldd; q.q = b.qd; q.s = b.sd; q.qt = b.qdt; q.st = b.sdt;
    q.colsum = a->need_db ? a->db : nullptr; q.colsum_part = b.part;
    const c1v_fp8_gemm_args gx = linear_gemm(b.qd, b.sd, b.qk, b.sk, a->rows, a->k, a->n, nullptr, a->x_dtype, a->dx, b);
    const c1v_fp8_gemm_args gk = linear_gemm(b.qxt, b.sxt, b.qdt, b.sdt, a->k, a->n, a->rows, nullptr, a->k_dtype, a->dk, b);
    if (a->need_dx && a->need_dk) {
        Fp8PairDev p{};
        Fp8Plan px, pk;
        if (gemm_setup(&gx, p.g[0], px) || gemm_setup(&gk, p.g[1], pk)) return -1;
        if (px.tile == 0 && pk.tile == 0 && px.splits == 1 && pk.splits == 1) {
            hipStream_t st = (hipStream_t)stream;
            if (quant_tiles(&q, nullptr, st, false)) return -1;
            for (Fp8GemmDev& g : p.g) { g.tiles_m = (int)c1v_cdiv(g.m, 64); g.tiles_n = (int)c1v_cdiv(g.n, 64); }
            p.blocks0 = p.g[0].tiles_m * p.g[0].tiles_n; p.blocks1 = p.g[1].tiles_m * p.g[1].tiles_n;
            p.part = b.part; p.tiles = c1v_cdiv(a->rows, FB); p.cols = a->n; p.sum = a->db;
            const unsigned blocks = (unsigned)(p.blocks0 + p.blocks1 + (a->need_db ? c1v_cdiv(a->n, 64) : 0));
            return launch_pair(p, blocks, st);
        }
    }
    int rc = c1v_fp8_quantize(&q, stream);
    if (!rc && a->need_dx) rc = c1v_fp8_gemm(&gx, stream);
    if (!rc && a->need_dk) rc = c1v_fp8_gemm(&gk, stream);
    return rc;
}
