// AdamW over many tensors at once, states in fp32 or in 8 bits.
//
//   g = f g            f = grad_scale, times (1 / |g|) clipnorm where |g| = |grad_scale| sqrt(sum g^2) is clipnorm or more
//   m' = b1 m + (1 - b1) g        v' = b2 v + (1 - b2) g^2
//   p' = (1 - lr wd) p - lr / (1 - b1^t) m' / (sqrt(v' / (1 - b2^t)) + eps)
//
// Bound by memory: 28 bytes a weight with fp32 states and gradients, 16 with 8-bit states (4 of p read and 4 written, 4 of g,
// 1 + 1 of each state and 4 bytes of scales per 128).  The clip reads g a second time, before (its norm is not known earlier).
// Measured, 160 M weights (a copy of 1 GiB reaches 5.1 TB/s): fp32 states 837 us = 5.3 TB/s; 8-bit states with bf16 gradients
// 422 us = 5.3 TB/s, with the clip 490 us: 92 for the norm (3.5 TB/s) and 395 for the update, which then finds some of g in the
// last-level cache.  8-bit states with parameters and gradients in bf16 355 us.  0.2 M weights in 12 tensors: 5.2 and 4 us.
//
// States in 8 bits.  A block of 128 elements shares a power-of-two scale for m and one for v; m is e4m3, v (never negative) a
// byte of five exponent and three mantissa bits.  Both are rounded STOCHASTICALLY from m' and v' in fp32 (the update uses the
// unrounded values): one step changes v by a thousandth, half a step of its byte is 3 to 6 hundredths, so rounding to nearest
// would hardly ever move it.  Rounded with the probability that the cut bits stand for, the held value follows in the mean.
// Powers of two for the scales keep the grid in place from step to step: what has not changed is held exactly, so the noise
// comes only with changes (a floating scale would throw the dice anew for every element in every step).  A v that is not zero
// never becomes zero: its square root divides.
#include "c1v_common.h"
#include "c1v_philox.h"

typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4_u __attribute__((ext_vector_type(4), aligned(2)));

constexpr int AW_CHUNK = C1V_ADAMW_CHUNK;           // 2048 elements per workgroup: 256 threads x 8
constexpr int AW_GROUP = C1V_ADAMW_GROUP;           // tensors per launch: their pointers travel in the kernel's arguments
constexpr int AW_PART = C1V_ADAMW_PARTIALS;         // workgroups of the norm pass per launch, at most
constexpr int AW_FEW = 256;                         // partial sums that every workgroup of the update adds up by itself

struct AdamwDev {
    const c1v_adamw_tensor* tab; int n_tab; int first, chunks, run;
    void* m; void* v; uint8_t* ms; uint8_t* vs;
    float b1, omb1, b2, omb2, eps, clipnorm, grad_scale; double lr_b1, lr_b2;
    int64_t* t; const double* lr; float* sched; double* part; int n_part, part0; float* norm; uint64_t* ctr; uint64_t seed;
    int lead;                                       // this launch moves the step on (norm pass) / writes the norm (update)
    int joined;                                     // the partial sums have been added up, the factor is in sched[3]
    uint32_t p_bf16[AW_GROUP / 32], g_bf16[AW_GROUP / 32];
    void* p[AW_GROUP]; const void* g[AW_GROUP];
};

__device__ __forceinline__ void load8(const void* base, int64_t i, int left, bool bf16, float* v) {
    if (!bf16) {
        const float* p = (const float*)base + i;
        if (left >= 8) {
            const f32x4_u a = *(const f32x4_u*)p, b = *(const f32x4_u*)(p + 4);
#pragma unroll
            for (int k = 0; k < 4; ++k) { v[k] = a[k]; v[4 + k] = b[k]; }
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = k < left ? p[k] : 0.f;
        }
    } else {
        const bf16_raw* p = (const bf16_raw*)base + i;
        if (left >= 8) {
            const u32x4_u a = *(const u32x4_u*)p;
#pragma unroll
            for (int k = 0; k < 4; ++k) { v[2 * k] = __uint_as_float(a[k] << 16); v[2 * k + 1] = __uint_as_float(a[k] & 0xffff0000u); }
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = k < left ? bf16_to_f32(p[k]) : 0.f;
        }
    }
}
__device__ __forceinline__ void store8(void* base, int64_t i, int left, bool bf16, const float* v) {
    if (!bf16) {
        float* p = (float*)base + i;
        if (left >= 8) {
            *(f32x4_u*)p = f32x4_u{v[0], v[1], v[2], v[3]};
            *(f32x4_u*)(p + 4) = f32x4_u{v[4], v[5], v[6], v[7]};
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) if (k < left) p[k] = v[k];
        }
    } else {                                        // parameters kept in bf16: rounded to nearest, off by half a step (2^-8)
        bf16_raw* p = (bf16_raw*)base + i;
        if (left >= 8) {
            *(u32x4_u*)p = u32x4_u{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) if (k < left) p[k] = f32_to_bf16(v[k]);
        }
    }
}
__device__ __forceinline__ bool bit(const uint32_t* a, int i) { return (a[i >> 5] >> (i & 31)) & 1; }

// index of the tensor that owns a chunk: the number of entries with first_chunk <= chunk, less one
__device__ __forceinline__ int tensor_of(const c1v_adamw_tensor* tab, int n, int chunk) {
    const int lane = threadIdx.x & 63;
    int found = 0;
    for (int b = 0; b < n; b += 64) {
        const int i = b + lane;
        found += __popcll(__ballot(i < n && tab[i].first_chunk <= chunk));
    }
    return found - 1;
}

// The workgroups of the norm pass take runs of d.run chunks in turn, so that at any time all of them work in one stretch of
// memory.  A run is walked tensor by tensor: tensor `ti`, described by T, owns the chunks up to `last`, `stop` is where it or
// the run ends.
struct ChunkWalk {
    const c1v_adamw_tensor* tab; int n_tab, len, run, c, run_end, end, ti, last, stop;
    c1v_adamw_tensor T;
    __device__ __forceinline__ ChunkWalk(const AdamwDev& d) : tab(d.tab), n_tab(d.n_tab), len(d.run) {
        end = d.first + d.chunks;
        run = c = d.first + min((int)blockIdx.x * len, d.chunks);
        run_end = min(c + len, end);
        ti = c < end ? tensor_of(tab, n_tab, c) : 0;
        enter();
    }
    __device__ __forceinline__ void enter() {
        T = tab[ti];
        last = ti + 1 < n_tab ? tab[ti + 1].first_chunk : end;
        stop = min(run_end, last);
    }
    __device__ __forceinline__ bool more() {                       // on to the tensor of chunk c (empty tensors own none)
        if (c >= run_end) {
            const int step = (int)gridDim.x * len;
            if (end - run <= step) return false;
            c = run += step;
            run_end = min(c + len, end);
            stop = min(run_end, last);
        }
        while (c >= last) { ++ti; enter(); }
        return true;
    }
};

// sum of squares in 64 bits, one partial sum per workgroup: the squares are exact and the order of the additions does not
// show in the fp32 norm, so that the clip factor (and through it the rounding of the 8-bit states) is reproducible anywhere
__global__ __launch_bounds__(256) void adamw_norm_kernel(AdamwDev d) {
    __shared__ double red[4];
    if (d.lead && blockIdx.x == 0 && threadIdx.x == 0) {
        const int64_t t = d.t[0] + 1;
        d.t[0] = t;
        d.sched[0] = (float)(d.lr[0] / (1.0 - pow(d.lr_b1, (double)t)));
        d.sched[1] = (float)(1.0 / (1.0 - pow(d.lr_b2, (double)t)));
        d.sched[2] = (float)d.lr[0];
        if (d.ctr) d.ctr[0] += 1;
    }
    if (d.clipnorm <= 0.f) return;
    double s = 0.0;
    ChunkWalk w(d);
    auto add = [&](const float* g) {
#pragma unroll
        for (int k = 0; k < 8; ++k) s = fma((double)g[k], (double)g[k], s);
    };
    while (w.more()) {
        const void* g = d.g[w.ti];
        const bool half = bit(d.g_bf16, w.ti);
        if (!g) { w.c = w.stop; continue; }
        int64_t i = (int64_t)(w.c - w.T.first_chunk) * AW_CHUNK + threadIdx.x * 8;
        for (; w.c + 4 <= w.stop && (int64_t)(w.c + 4 - w.T.first_chunk) * AW_CHUNK <= w.T.n; w.c += 4, i += 4 * AW_CHUNK) {
            float x[4][8];                                         // four chunks' loads in flight
#pragma unroll
            for (int q = 0; q < 4; ++q) load8(g, i + q * AW_CHUNK, 8, half, x[q]);
#pragma unroll
            for (int q = 0; q < 4; ++q) add(x[q]);
        }
        for (; w.c < w.stop; ++w.c, i += AW_CHUNK) {
            const int64_t left = w.T.n - i;
            if (left <= 0) continue;
            float x[8];
            load8(g, i, left > 8 ? 8 : (int)left, half, x);
            add(x);
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) d.part[d.part0 + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// The clip's factor (with grad_scale) from the partial sums of the norm; false: the step is left out, nothing moves.  `lead`
// writes the norm and takes the step number back.
__device__ __forceinline__ bool clip_factor(const AdamwDev& d, bool lead, float& f) {
    __shared__ double red[4];
    double s = 0.0;
    for (int i = threadIdx.x; i < d.n_part; i += 256) s += d.part[i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    const float norm = (float)sqrt((red[0] + red[1]) + (red[2] + red[3])) * fabsf(d.grad_scale);
    const bool fine = norm < __uint_as_float(0x7f800000u);                 // neither infinite nor NaN
    if (lead && threadIdx.x == 0) {
        d.norm[0] = norm;
        if (!fine) d.t[0] -= 1;
    }
    f = norm >= d.clipnorm ? ((1.0f / norm) * d.clipnorm) * d.grad_scale : d.grad_scale;
    return fine;
}
// many partial sums: added up once, before the update (in each of its workgroups they would cost more than its chunk)
__global__ __launch_bounds__(256) void adamw_join_kernel(AdamwDev d) {
    float f;
    const bool fine = clip_factor(d, true, f);
    if (threadIdx.x == 0) d.sched[3] = fine ? f : __uint_as_float(0x7fc00000u);
}

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t row_max(uint32_t v) {            // over the 16 lanes of a DPP row
    v = umax(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));
    v = umax(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));
    v = umax(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true));
    v = umax(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xF, 0xF, true));
    return v;
}
__device__ __forceinline__ float exp2_of(int s) { return __uint_as_float((uint32_t)s << 23); }        // 2^(s - 127), 1 <= s <= 254
__device__ __forceinline__ uint32_t finite_mag(float x) {
    const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
    return u >= 0x7f800000u ? 0u : u;
}

typedef float f32x2_t __attribute__((ext_vector_type(2)));

// The byte B of `w` <- e4m3 of m / scale; the largest magnitude of a block lies in [128, 256) of its scale, so rounding up cannot
// pass 448.  v_cvt_scalef32_sr_fp8_f32 adds the seed's upper 20 bits (16 random ones r, then 1000) to the 20 mantissa bits that
// are cut, so it carries with the probability they stand for.  Below the normal numbers, 2^-6, the value is first rounded to
// a multiple of 2^-29 (20 bits below a step), as the definition x + 2^-6 does.
template <int B> __device__ __forceinline__ uint32_t pack_m(uint32_t w, float m, float inv, uint32_t seed) {
    const float x = m * inv, c = copysignf(0x1p-6f, x);
    const float y = (x + c) - c;
    const float z = fabsf(x) < 0x1p-6f ? copysignf(y, x) : x;
    return (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(z, (int)seed, (int)w, B);
}
// v: byte c stands for the float with bits (c + 8 s - 240) << 20 (0: zero, 255: NaN); the block's largest value has c in 240 .. 248.
// base20 = (8 s - 240) << 20.  r2 = another 16 bits from the same r, shifted up by 4, plus 8.  Finite values only: they give eight
// bits, what is not finite would reach into its neighbours' bytes.
__device__ __forceinline__ uint32_t pack_v(float v, uint32_t base20, uint32_t r) {
    const uint32_t u = __float_as_uint(v), r2 = (__umul24(r, 40503u << 4) & 0xffff0u) | 8u;
    const int c = (int)(u + r2 - base20) >> 20, least = (int)(u < 1u ? u : 1u);      // 1 for what is not zero
    return (uint32_t)(c > least ? c : least);
}
__device__ __forceinline__ float unpack_v(uint32_t c, uint32_t base) { return c == 0 ? 0.f : __uint_as_float((c + base) << 20); }
__device__ __forceinline__ uint32_t has_ff(uint32_t w) { return (~w - 0x01010101u) & w & 0x80808080u; }       // some byte is 0xff

// One chunk per workgroup: the hardware hands them out in order, so that all CUs work in one stretch of memory, each at its own
// point of the way from loads to stores.  (160 M weights, fp32 / 8-bit states, us: 847 / 423 so; 896 / 458 with 2048 workgroups
// that take chunks in turn, 918 / 481 with a contiguous share for each.)
template <bool E8>
__global__ __launch_bounds__(256) void adamw_update_kernel(AdamwDev d) {
    float f = d.grad_scale;
    if (d.clipnorm > 0.f) {
        if (d.joined) {
            f = d.sched[3];
            if (f != f) return;
        } else if (!clip_factor(d, d.lead && blockIdx.x == 0, f)) return;
    }
    if ((int)blockIdx.x >= d.chunks) return;
    const float step = d.sched[0], ibc2 = d.sched[1], lr = d.sched[2];
    const int64_t t = d.t[0];
    const int c = d.first + (int)blockIdx.x, ti = __builtin_amdgcn_readfirstlane(tensor_of(d.tab, d.n_tab, c));
    const c1v_adamw_tensor T = d.tab[ti];
    if (!d.g[ti]) return;
    const int64_t i = (int64_t)(c - T.first_chunk) * AW_CHUNK + threadIdx.x * 8;
    if (i < ((T.n + 127) & ~(int64_t)127)) {                                // whole blocks of 128 = 16 lanes stay together
        const int64_t e = T.offset + i;
        const int64_t l64 = T.n - i;
        const int left = l64 > 8 ? 8 : (int)l64;
        const bool pb = bit(d.p_bf16, ti), gb = bit(d.g_bf16, ti);
        float g[8], p[8], m[8], v[8];
        load8(d.g[ti], i, left, gb, g);
        load8(d.p[ti], i, left, pb, p);
        if constexpr (E8) {
            const uint2 mq = *(const uint2*)((const uint8_t*)d.m + e), vq = *(const uint2*)((const uint8_t*)d.v + e);
            const float sm = exp2_of(d.ms[e >> 7]);
            const uint32_t base = 8u * d.vs[e >> 7] - 240u;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const f32x2_t x = k & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(k < 2 ? mq.x : mq.y, sm, true)
                                        : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(k < 2 ? mq.x : mq.y, sm, false);
                m[2 * k] = x[0]; m[2 * k + 1] = x[1];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = unpack_v(((k < 4 ? vq.x : vq.y) >> (8 * (k & 3))) & 0xff, base);
            if (__any((has_ff(vq.x) | has_ff(vq.y)) != 0)) {                 // a second moment that is no number
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if ((((k < 4 ? vq.x : vq.y) >> (8 * (k & 3))) & 0xff) == 0xff) v[k] = __uint_as_float(0x7fc00000u);
            }
        } else {
            const float4 a = *(const float4*)((const float*)d.m + e), b = *(const float4*)((const float*)d.m + e + 4);
            const float4 x = *(const float4*)((const float*)d.v + e), y = *(const float4*)((const float*)d.v + e + 4);
            m[0] = a.x; m[1] = a.y; m[2] = a.z; m[3] = a.w; m[4] = b.x; m[5] = b.y; m[6] = b.z; m[7] = b.w;
            v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
        }
        const float keep = 1.0f - lr * T.weight_decay, ibc2_up = ibc2 * 0x1p64f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
#pragma clang fp contract(off)
            const float gk = g[k] * f;                       // every operation rounded by itself: the moments, and with them
            const float a = m[k] * d.b1, b = gk * d.omb1;    // the 8-bit codes, do not depend on what a compiler fuses
            m[k] = a + b;
            const float q = gk * gk, x = v[k] * d.b2, y = q * d.omb2;
            v[k] = x + y;
            // square root and reciprocal to 1 ulp (v_sqrt_f32, v_rcp_f32): the update term is off by less than 2^-20 of itself.
            // v_sqrt_f32 takes denormal numbers for zero (an update of m / eps): small v are moved up by 2^64 before
            const bool low = v[k] < 0x1p-96f;
            const float den = __builtin_amdgcn_sqrtf(v[k] * (low ? ibc2_up : ibc2)) * (low ? 0x1p-32f : 1.f) + d.eps;
            p[k] = p[k] * keep - (m[k] * step) * __builtin_amdgcn_rcpf(den);
        }
        store8(d.p[ti], i, left, pb, p);
        if constexpr (E8) {
            uint32_t um = 0, uv = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) { um = umax(um, __float_as_uint(m[k]) & 0x7fffffffu); uv = umax(uv, __float_as_uint(v[k]) & 0x7fffffffu); }
            const bool odd = __any(umax(um, uv) >= 0x7f800000u);             // rare: only finite values make the scales
            uint32_t lost = 0;                                               // which v are no numbers (packed as 0, then marked)
            if (odd) {
                um = uv = 0;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    um = umax(um, finite_mag(m[k]));
                    if ((__float_as_uint(v[k]) & 0x7fffffffu) >= 0x7f800000u) { lost |= 1u << k; v[k] = 0.f; }
                    uv = umax(uv, __float_as_uint(v[k]));
                }
            }
            int sm = (int)(row_max(um) >> 23) - 7, sv = (int)(row_max(uv) >> 23);
            sm = sm < 1 ? 1 : sm;
            sv = sv < 32 ? 32 : sv;
            const uint64_t blk = (uint64_t)e >> 3;           // one Philox block gives the 16 random bits of eight elements
            const uint4 rnd = philox4x32_10(make_uint4((uint32_t)blk, (uint32_t)(blk >> 32), (uint32_t)t, (uint32_t)((uint64_t)t >> 32)), (uint32_t)d.seed, (uint32_t)(d.seed >> 32));
            const uint32_t rw[4] = {rnd.x, rnd.y, rnd.z, rnd.w};
            const float inv = exp2_of(254 - sm);
            const uint32_t base20 = (uint32_t)(8 * sv - 240) << 20;
            uint32_t mo[2] = {0, 0}, vo[2] = {0, 0};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                mo[h] = pack_m<0>(mo[h], m[4 * h], inv, (rw[2 * h] << 16) | 0x8000u);
                mo[h] = pack_m<1>(mo[h], m[4 * h + 1], inv, (rw[2 * h] & 0xffff0000u) | 0x8000u);
                mo[h] = pack_m<2>(mo[h], m[4 * h + 2], inv, (rw[2 * h + 1] << 16) | 0x8000u);
                mo[h] = pack_m<3>(mo[h], m[4 * h + 3], inv, (rw[2 * h + 1] & 0xffff0000u) | 0x8000u);
                vo[h] = pack_v(v[4 * h], base20, rw[2 * h] & 0xffffu) | pack_v(v[4 * h + 1], base20, rw[2 * h] >> 16) << 8 |
                        pack_v(v[4 * h + 2], base20, rw[2 * h + 1] & 0xffffu) << 16 | pack_v(v[4 * h + 3], base20, rw[2 * h + 1] >> 16) << 24;
            }
            if (odd) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const uint32_t sh = 8 * (k & 3);
                    if ((__float_as_uint(m[k]) & 0x7fffffffu) >= 0x7f800000u)
                        mo[k >> 2] = (mo[k >> 2] & ~(0xffu << sh)) | ((0x7fu | ((__float_as_uint(m[k]) >> 24) & 0x80u)) << sh);
                    if (lost >> k & 1) vo[k >> 2] |= 0xffu << sh;
                }
            }
            *(uint2*)((uint8_t*)d.m + e) = make_uint2(mo[0], mo[1]);
            *(uint2*)((uint8_t*)d.v + e) = make_uint2(vo[0], vo[1]);
            if ((threadIdx.x & 15) == 0) { d.ms[e >> 7] = (uint8_t)sm; d.vs[e >> 7] = (uint8_t)sv; }
        } else {
            *(float4*)((float*)d.m + e) = make_float4(m[0], m[1], m[2], m[3]);
            *(float4*)((float*)d.m + e + 4) = make_float4(m[4], m[5], m[6], m[7]);
            *(float4*)((float*)d.v + e) = make_float4(v[0], v[1], v[2], v[3]);
            *(float4*)((float*)d.v + e + 4) = make_float4(v[4], v[5], v[6], v[7]);
        }
    }
}

extern "C" int c1v_adamw_step(const c1v_adamw_args* a, void* stream) {
    C1V_REQUIRE(a && a->tensors && a->host && a->p && a->g && a->p_dtype && a->g_dtype && a->m && a->v && a->t && a->lr && a->sched && a->norm, "adamw_step: null argument");
    C1V_REQUIRE(a->n_tensors > 0 && a->n_tensors <= (1 << 20), "adamw_step: bad tensor count %d", a->n_tensors);
    C1V_REQUIRE(a->states == 0 || a->states == 1, "adamw_step: bad states %d", a->states);
    C1V_REQUIRE(a->states == 0 || (a->m_scale && a->v_scale), "adamw_step: 8-bit states need their scales");
    C1V_REQUIRE(((uintptr_t)a->m | (uintptr_t)a->v) % 16 == 0, "adamw_step: states must be 16-byte aligned");
    C1V_REQUIRE(a->beta1 >= 0 && a->beta1 < 1 && a->beta2 >= 0 && a->beta2 < 1, "adamw_step: betas must be in [0, 1)");
    C1V_REQUIRE(a->eps >= 1e-30f, "adamw_step: eps must be 1e-30 or more");
    const int groups = (a->n_tensors + AW_GROUP - 1) / AW_GROUP;
    C1V_REQUIRE(!(a->clipnorm > 0.f) || (a->partial && a->n_partial >= groups * AW_PART), "adamw_step: the clip needs %d partial sums", groups * AW_PART);
    int64_t chunk = a->host[0].first_chunk;
    for (int i = 0; i < a->n_tensors; ++i) {
        const c1v_adamw_tensor& t = a->host[i];
        C1V_REQUIRE(t.n >= 0 && t.offset >= 0 && t.offset % 128 == 0 && t.first_chunk == chunk, "adamw_step: bad table entry %d", i);
        chunk += c1v_cdiv(t.n, AW_CHUNK);
        C1V_REQUIRE(chunk < (1ll << 31) && chunk - a->host[i / AW_GROUP * AW_GROUP].first_chunk < (1ll << 24), "adamw_step: too many elements");
        C1V_REQUIRE(t.n == 0 || a->p[i], "adamw_step: tensor %d has no parameter", i);
        C1V_REQUIRE(a->p_dtype[i] <= C1V_BF16 && a->g_dtype[i] <= C1V_BF16, "adamw_step: bad dtype of tensor %d", i);
    }
    hipStream_t st = (hipStream_t)stream;
    AdamwDev d{};
    d.m = a->m; d.v = a->v; d.ms = (uint8_t*)a->m_scale; d.vs = (uint8_t*)a->v_scale;
    d.b1 = (float)a->beta1; d.omb1 = (float)(1.0 - a->beta1); d.b2 = (float)a->beta2; d.omb2 = (float)(1.0 - a->beta2);
    d.lr_b1 = a->beta1; d.lr_b2 = a->beta2; d.eps = a->eps; d.clipnorm = a->clipnorm; d.grad_scale = a->grad_scale;
    d.t = a->t; d.lr = a->lr; d.sched = a->sched; d.part = a->partial; d.norm = a->norm; d.ctr = a->ctr; d.seed = a->seed;
    for (int pass = 0; pass < 2; ++pass) {
        int parts = 0;
        d.joined = pass == 1 && a->clipnorm > 0.f && d.n_part > AW_FEW;
        if (d.joined) {
            hipLaunchKernelGGL(adamw_join_kernel, dim3(1), dim3(256), 0, st, d);
            C1V_LAUNCH_CHECK();
        }
        for (int k = 0; k < groups; ++k) {
            const int t0 = k * AW_GROUP, n = a->n_tensors - t0 < AW_GROUP ? a->n_tensors - t0 : AW_GROUP;
            const c1v_adamw_tensor& last = a->host[t0 + n - 1];
            d.tab = a->tensors + t0; d.n_tab = n; d.first = a->host[t0].first_chunk;
            d.chunks = last.first_chunk + (int)c1v_cdiv(last.n, AW_CHUNK) - d.first;
            for (int i = 0; i < AW_GROUP / 32; ++i) d.p_bf16[i] = d.g_bf16[i] = 0;
            for (int i = 0; i < n; ++i) {
                d.p[i] = a->p[t0 + i]; d.g[i] = a->g[t0 + i];
                if (a->p_dtype[t0 + i] == C1V_BF16) d.p_bf16[i >> 5] |= 1u << (i & 31);
                if (a->g_dtype[t0 + i] == C1V_BF16) d.g_bf16[i >> 5] |= 1u << (i & 31);
            }
            d.lead = k == 0;
            if (pass == 0) {
                const bool clip = a->clipnorm > 0.f;
                if (!clip && k > 0) break;
                // few chunks: up to AW_FEW workgroups, whose sums the update adds up itself; many: up to AW_PART, eight chunks at a time
                // (160 M weights, bf16 gradients, what the clip adds to a step: 71 us; 2048 workgroups with a share each 86, four
                // chunks at a time 88)
                d.run = (int)c1v_cdiv(d.chunks, AW_FEW);
                d.run = d.run < 1 ? 1 : d.run > 8 ? 8 : d.run;
                const int runs = (int)c1v_cdiv(d.chunks, d.run);
                const int grid = !clip || runs < 1 ? 1 : runs < AW_PART ? runs : AW_PART;
                d.part0 = parts;
                parts += grid;
                hipLaunchKernelGGL(adamw_norm_kernel, dim3((unsigned)grid), dim3(256), 0, st, d);
                C1V_LAUNCH_CHECK();
                d.n_part = parts;
            } else {
                if (d.chunks < 1 && !d.lead) continue;
                const int grid = d.chunks < 1 ? 1 : d.chunks;
                if (a->states == 1) hipLaunchKernelGGL(adamw_update_kernel<true>, dim3((unsigned)grid), dim3(256), 0, st, d);
                else hipLaunchKernelGGL(adamw_update_kernel<false>, dim3((unsigned)grid), dim3(256), 0, st, d);
                C1V_LAUNCH_CHECK();
            }
        }
    }
    return 0;
}
