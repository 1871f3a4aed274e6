// The AdamW step over many tensors at once, and the global norm of their gradients:
//
//   g' = g c            c = min(1, max_norm / (|g| + 1e-6)), |g| over all tensors; 1 without a limit
//   m' = b1 m + (1 - b1) g'
//   v' = b2 v + (1 - b2) g'^2
//   p' = (1 - lr wd) p - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// One launch steps up to kMaxTensors tensors: their addresses travel in the kernel's own
// parameters (no table on the device to upload or keep), the tensors are cut into chunks of
// kChunk elements, and every block takes an equal run of them: it searches for its first tensor
// once, then goes from one to the next.
//
// 8-bit moments: kQ = 256 elements share a float scale, their largest finite magnitude over
// 448, and each is an e4m3 code (3 fraction bits). The moments are moving averages: a step
// moves m by a tenth and v by a thousandth of the way, less than half of the format's spacing
// (6-12%), so rounding to nearest would leave them standing; the codes are rounded up with
// the probability of the part dropped instead, the random bits a hash of the step, the seed
// and the element's number. A v above zero is never held as zero (its root divides), unless its
// block's largest is below 1e-30: such blocks are held as zeros.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <math_constants.h>

#include <cmath>
#include <cstddef>

#include "common.cuh"

namespace wt {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 2048;  // elements of one work item: a block of kQ for each warp
constexpr int kQ = WT_ADAMW_BLOCK;
constexpr int kMaxTensors = 320;  // of one launch: the table stays below the 32,764 bytes a kernel's parameters may have
constexpr int kFewTensors = 24;

// What a launch knows of a tensor. first: the number of its first element among all of the
// optimiser's, each tensor starting on a whole block of kQ. before: the steps before the tensor's
// first, or null. keep: 1 - lr wd. wide: its operands allow access to four elements at once (16
// bytes, of all of them with 8-bit moments).
struct __align__(16) Row {
    void *p;
    const void *g;
    void *m, *v;
    float *m_scale, *v_scale, *master;
    long long numel;
    unsigned long long first;
    const long long *before;
    float lr, keep;
    int wide, type;
};

template <int MAX>
struct Table {
    Row row[MAX];
    unsigned chunk[MAX + 1];  // chunks before each tensor
    int n;
};

// The table as memory that is loaded through the data cache: reads of the constant bank by an index
// that varies cost some microseconds a block (150 tensors, 60 MB: 37 us for their norm).
template <int MAX>
__device__ __forceinline__ const Table<MAX> *as_memory(const Table<MAX> &tb) {
    const Table<MAX> *p = &tb;
    asm volatile("" : "+l"(p));
    return p;
}

struct Step {
    float b1, c1, b2, c2, eps, minus_zero;
    float corr1, corr2;    // 1 / (1 - b1^t), 1 / sqrt(1 - b2^t) of tensors without `before` when `skipped` is null
    float log_b1, log_b2;  // else t - *skipped - *before takes the place of t
    long long t;
    const WtStepControl *control;
    const long long *skipped;
    unsigned key0, key1;
};

__device__ __forceinline__ float load(const float *p) { return *p; }
__device__ __forceinline__ float load(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load(const __half *p) { return __half2float(*p); }
__device__ __forceinline__ void store(float *p, float x) { *p = x; }
__device__ __forceinline__ void store(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void store(__half *p, float x) { *p = __float2half_rn(x); }

// Four adjacent elements, aligned to their size.
__device__ __forceinline__ float4 load4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16 *p) {
    const uint2 q = *reinterpret_cast<const uint2 *>(p);
    return make_float4(__uint_as_float(q.x << 16), __uint_as_float(q.x & 0xFFFF0000u), __uint_as_float(q.y << 16),
                       __uint_as_float(q.y & 0xFFFF0000u));
}
__device__ __forceinline__ float4 load4(const __half *p) {
    const uint2 q = *reinterpret_cast<const uint2 *>(p);
    const float2 u = __half22float2(reinterpret_cast<const __half2 &>(q.x)), v = __half22float2(reinterpret_cast<const __half2 &>(q.y));
    return make_float4(u.x, u.y, v.x, v.y);
}
__device__ __forceinline__ void store4(float *p, float4 x) { *reinterpret_cast<float4 *>(p) = x; }
__device__ __forceinline__ void store4(__nv_bfloat16 *p, float4 x) {
    const __nv_bfloat162 u = __floats2bfloat162_rn(x.x, x.y), v = __floats2bfloat162_rn(x.z, x.w);
    *reinterpret_cast<uint2 *>(p) = make_uint2(reinterpret_cast<const unsigned &>(u), reinterpret_cast<const unsigned &>(v));
}
__device__ __forceinline__ void store4(__half *p, float4 x) {
    const __half2 u = __floats2half2_rn(x.x, x.y), v = __floats2half2_rn(x.z, x.w);
    *reinterpret_cast<uint2 *>(p) = make_uint2(reinterpret_cast<const unsigned &>(u), reinterpret_cast<const unsigned &>(v));
}

// The equal run of block `block` of a launch's chunks, tensor by tensor: body(row, first element, end).
template <int MAX, typename Body>
__device__ __forceinline__ void run_of_chunks(const Table<MAX> &table, unsigned block, Body body) {
    const Table<MAX> *tb = as_memory(table);
    const int n = table.n, lane = threadIdx.x & 31;
    const unsigned long long chunks = tb->chunk[n];
    unsigned c = (unsigned)(chunks * block / gridDim.x);
    const unsigned stop = (unsigned)(chunks * (block + 1) / gridDim.x);
    if (c == stop) return;
    // the last tensor whose first chunk is not after c: by the warp, every kEach-th tensor, then those between
    constexpr int kEach = (MAX + 31) / 32;
    int k = 0;
    if (kEach > 1) {
        const int at = lane * kEach;
        k = (31 - __clz(__ballot_sync(kFull, at < n && tb->chunk[at] <= c))) * kEach;
    }
    const int at = k + lane;
    k += 31 - __clz(__ballot_sync(kFull, at < n && (kEach == 1 || lane < kEach) && tb->chunk[at] <= c));
    for (; c < stop; k++) {
        const unsigned first = tb->chunk[k], end = min(stop, tb->chunk[k + 1]);
        if (end <= c) continue;  // a tensor of no elements
        const Row &row = table.row[k];
        body(row, (long long)(c - first) * kChunk, min((long long)(end - first) * kChunk, row.numel));
        c = end;
    }
}

__device__ __forceinline__ unsigned mix(unsigned z, unsigned k0, unsigned k1) {
    z ^= k0;
    z ^= z >> 16;
    z *= 0x6A09E667u;  // odd 32-bit fractions of the square roots of 2 and 3
    z ^= z >> 15;
    z ^= k1;
    z *= 0xBB67AE85u;
    return z ^ (z >> 16);
}

// y (|y| <= 448 up to rounding) rounded to a value of e4m3 by 16 random bits: the 20 fraction
// bits that the format drops are compared with them by adding them in and cutting. Below 2^-6,
// where the format's spacing is even (2^-9), 2^-6 is added first, which puts that spacing at the
// same bit. The four steps: small_of(y); y + small; cut(that, 16 r + 8); that - small.
template <bool POSITIVE>
__device__ __forceinline__ float small_of(float y) {
    return POSITIVE ? (y < 0.015625f ? 0.015625f : 0.0f) : fabsf(y) < 0.015625f ? copysignf(0.015625f, y) : 0.0f;
}
__device__ __forceinline__ float cut(float y, unsigned bits) { return __uint_as_float((__float_as_uint(y) + bits) & 0xFFF00000u); }

__device__ __forceinline__ unsigned char encode(float z) { return __nv_cvt_float_to_fp8(z, __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ float decode(unsigned char code) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(code, __NV_E4M3)));
}

// Four codes of a word.
__device__ __forceinline__ unsigned encode4(const float (&z)[4]) {
    const unsigned lo = __nv_cvt_float2_to_fp8x2(make_float2(z[0], z[1]), __NV_SATFINITE, __NV_E4M3);
    const unsigned hi = __nv_cvt_float2_to_fp8x2(make_float2(z[2], z[3]), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}
__device__ __forceinline__ void decode4(unsigned word, float (&x)[4]) {
    const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(word & 0xFFFFu), __NV_E4M3);
    const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(word >> 16), __NV_E4M3);
    const float2 a = __half22float2(__half2(lo)), b = __half22float2(__half2(hi));
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}

// Behind a norm the last gradients go first: they are still in L2.
__device__ __forceinline__ unsigned block_of(const Step &s) { return s.control ? gridDim.x - 1 - blockIdx.x : blockIdx.x; }

struct Rates {
    float clip, corr1, corr2;
};

// False when the step is to be left out (the norm was not finite).
__device__ __forceinline__ bool clip_of(const Step &s, float &clip) {
    clip = s.control ? s.control->clip : 1.0f;
    return !s.control || !s.control->skip;
}

__device__ __forceinline__ Rates rates_of(const Row &row, const Step &s, float clip) {
    if (!s.skipped && !row.before) return Rates{clip, s.corr1, s.corr2};
    const float t = (float)(s.t - (s.skipped ? *s.skipped : 0) - (row.before ? *row.before : 0));
    return Rates{clip, 1.0f / -expm1f(t * s.log_b1), rsqrtf(-expm1f(t * s.log_b2))};
}

// The root and the reciprocal are the hardware's (one and two units in the last place): an error
// of 2^-22 of the step, far below the parameter's own rounding; the moments do not depend on it.
__device__ __forceinline__ float updated(float p, float m, float v, float keep, float rate, float corr2, float eps) {
    float root, inv;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(root) : "f"(v));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(__fmaf_rn(root, corr2, eps)));
    return __fmaf_rn(p, keep, -rate * (m * inv));
}

// Two floats in one register pair: one instruction does both (each result rounded on its own).
struct Two {
    unsigned long long bits;
    __device__ __forceinline__ Two() {}
    __device__ __forceinline__ Two(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(bits) : "f"(x), "f"(y)); }
    __device__ __forceinline__ void get(float &x, float &y) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(bits)); }
};
__device__ __forceinline__ Two operator*(Two a, Two b) {
    Two r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
    return r;
}
__device__ __forceinline__ Two operator+(Two a, Two b) {
    Two r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits));
    return r;
}
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
    return r;
}
__device__ __forceinline__ Two both(float x) { return Two(x, x); }

// One element's moments: each product and sum rounded on its own, so that what is held in 8 bits
// follows from its inputs alone.
__device__ __forceinline__ void advance(float g, float &m, float &v, const Step &s) {
    m = m * s.b1 + g * s.c1;
    v = v * s.b2 + (g * g) * s.c2;
}

// 32-bit moments, bound by memory: 28 bytes an element, each once. 46M float weights 200 us, 6.4 TB/s;
// 150 bf16 tensors of 30M elements 131 us, 6.4 TB/s.
template <typename P, int MAX>
__global__ void __launch_bounds__(kThreads, 5) adamw32(const __grid_constant__ Table<MAX> tb, const __grid_constant__ Step s) {
    float clip;
    if (!clip_of(s, clip)) return;
    run_of_chunks(tb, block_of(s), [&](const Row &t, long long first, long long end) {
        const Rates r = rates_of(t, s, clip);
        constexpr bool kMaster = sizeof(P) == 2;
        P *const p = static_cast<P *>(t.p);
        const P *const g = static_cast<const P *>(t.g);
        float *const m = static_cast<float *>(t.m), *const v = static_cast<float *>(t.v);
        float *const master = kMaster ? t.master : reinterpret_cast<float *>(p);
        const float rate = t.lr * r.corr1, keep = t.keep;
        auto one = [&](float p, float g, float &m, float &v) {
            advance(g * r.clip, m, v, s);
            return updated(p, m, v, keep, rate, r.corr2, s.eps);
        };
        long long single = first;
        if (t.wide) {
            single = end & ~3LL;
#pragma unroll 2
            for (long long j = first + threadIdx.x * 4; j < single; j += kThreads * 4) {
                float4 gj = load4(g + j), mj = load4(m + j), vj = load4(v + j), pj = load4(master + j);
                pj.x = one(pj.x, gj.x, mj.x, vj.x);
                pj.y = one(pj.y, gj.y, mj.y, vj.y);
                pj.z = one(pj.z, gj.z, mj.z, vj.z);
                pj.w = one(pj.w, gj.w, mj.w, vj.w);
                store4(m + j, mj);
                store4(v + j, vj);
                store4(master + j, pj);
                if (kMaster) store4(p + j, pj);
            }
        }
        for (long long j = single + threadIdx.x; j < end; j += kThreads) {
            float mj = m[j], vj = v[j];
            const float pj = one(master[j], load(g + j), mj, vj);
            m[j] = mj;
            v[j] = vj;
            master[j] = pj;
            if (kMaster) store(p + j, pj);
        }
    });
}

// What a warp reads of a block of kQ elements.
template <typename P>
struct Operands {
    const float *master;
    const P *g;
    const unsigned char *m, *v;
    float ms, vs;
};

// A warp per block of kQ elements, eight elements a thread: two runs of four adjacent ones where
// the operands allow it (WIDE), else single ones 32 apart. 70 instructions an element against 16
// bytes, some 20 of them the hash and the rounding: issuing them takes as long as the memory, so
// pairs of floats go through the packed instructions (81 without). 300M weights 0.87 ms, 5.5 TB/s,
// instructions issued in 68% of the cycles.
template <bool WIDE, typename P>
__device__ __forceinline__ void adamw8_block(const Operands<P> &in, P *p, unsigned char *m, unsigned char *v, float *master,
                                             float *m_scale, float *v_scale, int n, unsigned hash, float keep, float rate,
                                             const Rates &r, const Step &s) {
    constexpr bool kMaster = sizeof(P) == 2;
    const int lane = threadIdx.x & 31;
    auto place = [&](int j) { return WIDE ? (j & 4) * 32 + lane * 4 + (j & 3) : j * 32 + lane; };
    float mj[8], vj[8], pj[8], gj[8];
    if (WIDE) {
#pragma unroll
        for (int h = 0; h < 8; h += 4) {
            const int at = place(h);
            const float4 a = load4(in.master + at), b = load4(in.g + at);
            const unsigned mw = *reinterpret_cast<const unsigned *>(in.m + at), vw = *reinterpret_cast<const unsigned *>(in.v + at);
            pj[h] = a.x, pj[h + 1] = a.y, pj[h + 2] = a.z, pj[h + 3] = a.w;
            gj[h] = b.x, gj[h + 1] = b.y, gj[h + 2] = b.z, gj[h + 3] = b.w;
            decode4(mw, reinterpret_cast<float(&)[4]>(mj[h]));
            decode4(vw, reinterpret_cast<float(&)[4]>(vj[h]));
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int at = place(j);
            const bool there = at < n;
            pj[j] = there ? in.master[at] : 0.0f;
            gj[j] = there ? load(in.g + at) : 0.0f;
            mj[j] = there ? decode(in.m[at]) : 0.0f;
            vj[j] = there ? decode(in.v[at]) : 0.0f;
        }
    }
    const float ms = in.ms, vs = in.vs;
    unsigned mtop = 0, vtop = 0;  // largest magnitudes, as bits: what is not a number is the largest of all
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const Two x = Two(gj[j], gj[j + 1]) * both(r.clip);
        // as `advance`: a packed product that a sum takes would be contracted with it, a sum of the
        // product and the -0 the host gives is not
        const Two zero = both(s.minus_zero);
        const Two m2 = fma(Two(mj[j], mj[j + 1]) * both(ms), both(s.b1), zero) + fma(x, both(s.c1), zero);
        const Two v2 = fma(Two(vj[j], vj[j + 1]) * both(vs), both(s.b2), zero) + fma(x * x, both(s.c2), zero);
        m2.get(mj[j], mj[j + 1]);
        v2.get(vj[j], vj[j + 1]);
        float root[2], inv[2];
#pragma unroll
        for (int i = 0; i < 2; i++) asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(root[i]) : "f"(vj[j + i]));
        fma(Two(root[0], root[1]), both(r.corr2), both(s.eps)).get(root[0], root[1]);
#pragma unroll
        for (int i = 0; i < 2; i++) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv[i]) : "f"(root[i]));
        const Two step = (m2 * Two(inv[0], inv[1])) * both(-rate);
        fma(Two(pj[j], pj[j + 1]), both(keep), step).get(pj[j], pj[j + 1]);
#pragma unroll
        for (int i = j; i < j + 2; i++) {
            mtop = max(mtop, __float_as_uint(mj[i]) & 0x7FFFFFFFu);
            vtop = max(vtop, __float_as_uint(vj[i]));
        }
    }
    if (WIDE) {
#pragma unroll
        for (int h = 0; h < 8; h += 4) {
            const float4 q = make_float4(pj[h], pj[h + 1], pj[h + 2], pj[h + 3]);
            store4(master + place(h), q);
            if (kMaster) store4(p + place(h), q);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int at = place(j);
            if (at < n) {
                master[at] = pj[j];
                if (kMaster) store(p + at, pj[j]);
            }
        }
    }
    mtop = __reduce_max_sync(kFull, mtop);
    vtop = __reduce_max_sync(kFull, vtop);
    unsigned odd = 0;  // elements that are not finite: held as NaN, e4m3 having no infinity, and no part of the scale
    if (max(mtop, vtop) >= 0x7F800000u) {
        mtop = vtop = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const unsigned mb = __float_as_uint(mj[j]) & 0x7FFFFFFFu, vb = __float_as_uint(vj[j]) & 0x7FFFFFFFu;
            if (mb >= 0x7F800000u) odd |= 1u << j;
            else mtop = max(mtop, mb);
            if (vb >= 0x7F800000u) odd |= 256u << j;
            else vtop = max(vtop, vb);
        }
        mtop = __reduce_max_sync(kFull, mtop);
        vtop = __reduce_max_sync(kFull, vtop);
    }
    // one division for both: the lanes of an odd number take v's
    const float top = __uint_as_float(lane & 1 ? vtop : mtop), inv = top >= 1e-30f ? (1.0f / top) * 448.0f : 0.0f;
    const float minv = __shfl_sync(kFull, inv, 0), vinv = __shfl_sync(kFull, inv, 1);
    if (lane == 0) {
        *m_scale = minv > 0.0f ? __uint_as_float(mtop) * (1.0f / 448.0f) : 0.0f;
        *v_scale = vinv > 0.0f ? __uint_as_float(vtop) * (1.0f / 448.0f) : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const Two zero = both(s.minus_zero), minus = both(-1.0f);
        const Two my = fma(Two(mj[j], mj[j + 1]), both(minv), zero), vy = fma(Two(vj[j], vj[j + 1]), both(vinv), zero);
        float y[2], ms[2], vs[2], m[2], v[2];
        my.get(y[0], y[1]);
        ms[0] = small_of<false>(y[0]), ms[1] = small_of<false>(y[1]);
        vy.get(y[0], y[1]);
        vs[0] = small_of<true>(y[0]), vs[1] = small_of<true>(y[1]);
        (my + Two(ms[0], ms[1])).get(m[0], m[1]);
        (vy + Two(vs[0], vs[1])).get(v[0], v[1]);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            // the number is that of a whole block of kQ with the place in its low bits
            const unsigned z = mix(hash ^ (unsigned)place(j + i), s.key0, s.key1);
            m[i] = cut(m[i], (z << 4 & 0xFFFF0u) | 8u);
            v[i] = cut(v[i], (z >> 12 & 0xFFFF0u) | 8u);
        }
        fma(Two(ms[0], ms[1]), minus, Two(m[0], m[1])).get(mj[j], mj[j + 1]);
        fma(Two(vs[0], vs[1]), minus, Two(v[0], v[1])).get(vj[j], vj[j + 1]);
#pragma unroll
        for (int i = 0; i < 2; i++)
            if (y[i] > 0.0f) vj[j + i] = fmaxf(vj[j + i], 0.001953125f);
    }
    if (odd) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (odd >> j & 1) mj[j] = CUDART_NAN_F;
            if (odd >> j & 256) vj[j] = CUDART_NAN_F;
        }
    }
    if (WIDE) {
#pragma unroll
        for (int h = 0; h < 8; h += 4) {
            *reinterpret_cast<unsigned *>(m + place(h)) = encode4(reinterpret_cast<float(&)[4]>(mj[h]));
            *reinterpret_cast<unsigned *>(v + place(h)) = encode4(reinterpret_cast<float(&)[4]>(vj[h]));
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int at = place(j);
            if (at < n) {
                m[at] = encode(mj[j]);
                v[at] = encode(vj[j]);
            }
        }
    }
}

// A block of kQ elements' operands in shared memory, on their way while the warp works on another.
template <typename P>
struct __align__(16) Slot {
    float master[kQ];
    P g[kQ];
    unsigned char m[kQ], v[kQ];
    static __device__ __forceinline__ void copy16(void *to, const void *from) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from) : "memory");
    }
    __device__ __forceinline__ void fetch(const float *master_at, const P *g_at, const unsigned char *m_at, const unsigned char *v_at) {
        constexpr int kG = 16 / sizeof(P);
        const int lane = threadIdx.x & 31;
        copy16(master + lane * 4, master_at + lane * 4);
        copy16(master + kQ / 2 + lane * 4, master_at + kQ / 2 + lane * 4);
        copy16(g + lane * kG, g_at + lane * kG);
        if (sizeof(P) == 4) copy16(g + kQ / 2 + lane * kG, g_at + kQ / 2 + lane * kG);
        copy16((lane < 16 ? m : v) + lane % 16 * 16, (lane < 16 ? m_at : v_at) + lane % 16 * 16);
    }
};

template <typename P, int MAX>
__global__ void __launch_bounds__(kThreads, 4) adamw8(const __grid_constant__ Table<MAX> tb, const __grid_constant__ Step s) {
    __shared__ Slot<P> slots[kThreads / 32][2];
    float clip;
    if (!clip_of(s, clip)) return;
    run_of_chunks(tb, block_of(s), [&](const Row &t, long long first, long long end) {
        const Rates r = rates_of(t, s, clip);
        P *const p = static_cast<P *>(t.p);
        float *const master = sizeof(P) == 2 ? t.master : reinterpret_cast<float *>(p);
        const P *const g = static_cast<const P *>(t.g);
        unsigned char *const m = static_cast<unsigned char *>(t.m), *const v = static_cast<unsigned char *>(t.v);
        float *const ms = t.m_scale, *const vs = t.v_scale;
        const unsigned long long number = t.first;
        const float rate = t.lr * r.corr1, keep = t.keep;
        constexpr int kStride = kThreads / 32 * kQ;
        Slot<P> *const slot = slots[threadIdx.x >> 5];
        long long at = first + (threadIdx.x >> 5) * kQ;
        auto hash_of = [&](long long at) {
            const unsigned long long i = number + at;
            return (unsigned)i ^ (unsigned)(i >> 32) * 0x9E3779B1u;
        };
        if (t.wide) {
            float ms_next = 0.0f, vs_next = 0.0f;
            auto fetch = [&](long long at, int to) {
                if (at + kQ <= end) {
                    slot[to].fetch(master + at, g + at, m + at, v + at);
                    ms_next = ms[at / kQ], vs_next = vs[at / kQ];
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            __syncwarp();  // the tensor before is done with the slots
            fetch(at, 0);
            for (int parity = 0; at + kQ <= end; at += kStride, parity ^= 1) {
                Operands<P> in{slot[parity].master, slot[parity].g, slot[parity].m, slot[parity].v, ms_next, vs_next};
                __syncwarp();  // all have read what is fetched over
                fetch(at + kStride, parity ^ 1);
                asm volatile("cp.async.wait_group 1;" ::: "memory");
                __syncwarp();  // all lanes' copies are here
                adamw8_block<true>(in, p + at, m + at, v + at, master + at, ms + at / kQ, vs + at / kQ, kQ, hash_of(at), keep, rate, r, s);
            }
        }
        for (; at < end; at += kStride) {
            const Operands<P> in{master + at, g + at, m + at, v + at, ms[at / kQ], vs[at / kQ]};
            adamw8_block<false>(in, p + at, m + at, v + at, master + at, ms + at / kQ, vs + at / kQ, (int)min((long long)kQ, end - at),
                                hash_of(at), keep, rate, r, s);
        }
    });
}

// The sum of squares of elements [first, end), a float over at most 64 of a thread's, then double.
template <typename P>
__device__ __forceinline__ double square_sum(const void *data, long long first, long long end, bool wide) {
    const P *const g = static_cast<const P *>(data);
    double sum = 0.0;
    long long single = first;
    if (wide) {
        single = end & ~3LL;
        constexpr int kBatch = 8;  // loads of a thread on their way at once
        long long i = first + threadIdx.x * 4;
        for (; i + (kBatch - 1) * kThreads * 4 < single; i += kBatch * kThreads * 4) {
            float4 x[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; k++) x[k] = load4(g + i + k * kThreads * 4);
            float a = 0.0f, b = 0.0f, c = 0.0f, d = 0.0f;
#pragma unroll
            for (int k = 0; k < kBatch; k++) {
                a = __fmaf_rn(x[k].x, x[k].x, a);
                b = __fmaf_rn(x[k].y, x[k].y, b);
                c = __fmaf_rn(x[k].z, x[k].z, c);
                d = __fmaf_rn(x[k].w, x[k].w, d);
            }
            sum += (double)((a + b) + (c + d));
        }
        float a = 0.0f;
        for (; i < single; i += kThreads * 4) {
            const float4 x = load4(g + i);
            a += __fmaf_rn(x.x, x.x, x.y * x.y) + __fmaf_rn(x.z, x.z, x.w * x.w);
        }
        sum += (double)a;
    }
    float a = 0.0f;
    int taken = 0;
    for (long long i = single + threadIdx.x; i < end; i += kThreads) {
        const float x = load(g + i);
        a = __fmaf_rn(x, x, a);
        if (++taken == 64) {
            sum += (double)a;
            a = 0.0f;
            taken = 0;
        }
    }
    return sum + (double)a;
}

// One float64 partial per block, joined in their order by the block that arrives last. Squares are
// float's: a gradient above 1.8e19 makes the norm infinite. 46M float
// gradients 37 us, 5.0 TB/s (some 6 us of it the last block's part).
template <int MAX>
__global__ void __launch_bounds__(kThreads, 4) norm_kernel(const __grid_constant__ Table<MAX> tb, double *partial, unsigned blocks,
                                                        unsigned before, float max_norm, WtStepControl *control) {
    __shared__ double part[kThreads / 32];
    __shared__ bool last;
    double sum = 0.0;
    run_of_chunks(tb, blockIdx.x, [&](const Row &t, long long first, long long end) {
        sum += t.type == WT_F32    ? square_sum<float>(t.g, first, end, t.wide)
               : t.type == WT_BF16 ? square_sum<__nv_bfloat16>(t.g, first, end, t.wide)
                                       : square_sum<__half>(t.g, first, end, t.wide);
    });
    auto block_sum = [&](double v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_down_sync(kFull, v, o);
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
        __syncthreads();
        double tot = 0.0;
        for (int w = 0; w < kThreads / 32; w++) tot += part[w];
        __syncthreads();
        return tot;
    };
    const double tot = block_sum(sum);
    if (threadIdx.x == 0) {
        partial[before + blockIdx.x] = tot;
        __threadfence();
        last = atomicAdd(&control->arrived, 1u) == blocks - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    double all = 0.0;
    for (unsigned i = threadIdx.x; i < blocks; i += kThreads) all += __ldcg(partial + i);
    all = block_sum(all);
    if (threadIdx.x == 0) {
        const float norm = (float)sqrt(all);
        const bool fine = isfinite(norm);
        control->arrived = 0;
        control->norm = norm;
        control->clip = max_norm > 0.0f ? fminf(1.0f, max_norm / (norm + 1e-6f)) : 1.0f;
        control->skip = !fine;
        if (!fine) control->skipped += 1;
    }
}

// Blocks of a launch: a chunk each while they are few, then eight rounds of four blocks an SM, none
// with a shorter run than eight chunks. Several rounds, since with one the launch waits for its
// slowest run (46M float weights: 215 us with 8 blocks an SM, 205 with 16, 200 with 32).
constexpr unsigned kFew = 148 * 8, kMany = 148 * 32;
unsigned blocks_for(long long chunks) {
    if (chunks <= kFew) return chunks < 1 ? 1 : (unsigned)chunks;
    const long long blocks = chunks / 8;
    return blocks < kFew ? kFew : blocks < kMany ? (unsigned)blocks : kMany;
}

bool aligned(uint64_t p, int to) { return p % to == 0; }

unsigned chunks_of(int64_t numel) { return (unsigned)((numel + kChunk - 1) / kChunk); }

// The table of tensors [from, from + n) of a call.
template <int MAX>
void fill(Table<MAX> &tb, const WtAdamW &a, int from, int n) {
    unsigned chunks = 0;
    tb.n = n;
    const int z = a.type == WT_F32 || a.state_bits == 8 ? 16 : 8;
    for (int i = 0; i < n; i++) {
        const int k = from + i;
        Row &t = tb.row[i];
        t.p = (void *)a.p[k];
        t.g = (const void *)a.g[k];
        t.m = (void *)a.m[k];
        t.v = (void *)a.v[k];
        t.m_scale = a.m_scale ? (float *)a.m_scale[k] : nullptr;
        t.v_scale = a.v_scale ? (float *)a.v_scale[k] : nullptr;
        t.master = a.master ? (float *)a.master[k] : nullptr;
        t.numel = a.numel[k];
        t.first = a.first ? (unsigned long long)a.first[k] : 0;
        t.before = a.before ? (const long long *)a.before[k] : nullptr;
        t.lr = (float)a.lr[k];
        t.keep = (float)(1.0 - a.lr[k] * a.weight_decay[k]);
        t.type = a.type;
        t.wide = aligned(a.p[k], z) && aligned(a.g[k], z) && aligned(a.m[k], 16) && aligned(a.v[k], 16) &&
                 (!a.master || aligned(a.master[k], 16));
        tb.chunk[i] = chunks;
        chunks += chunks_of(a.numel[k]);
    }
    tb.chunk[n] = chunks;
}

unsigned mix_host(unsigned z, unsigned k0, unsigned k1) {
    z ^= k0;
    z ^= z >> 16;
    z *= 0x6A09E667u;
    z ^= z >> 15;
    z ^= k1;
    z *= 0xBB67AE85u;
    return z ^ (z >> 16);
}

Step step_of(const WtAdamW &a) {
    Step s{};
    s.b1 = (float)a.beta1;
    s.c1 = (float)(1.0 - a.beta1);
    s.b2 = (float)a.beta2;
    s.c2 = (float)(1.0 - a.beta2);
    s.eps = (float)a.eps;
    s.minus_zero = -0.0f;
    s.corr1 = (float)(1.0 / (1.0 - std::pow(a.beta1, (double)a.step)));
    s.corr2 = (float)(1.0 / std::sqrt(1.0 - std::pow(a.beta2, (double)a.step)));
    s.log_b1 = (float)std::log(a.beta1);
    s.log_b2 = (float)std::log(a.beta2);
    s.t = a.step;
    s.control = a.control;
    if (a.skipped) s.skipped = (const long long *)a.skipped;
    else if (a.control) s.skipped = (const long long *)((const char *)a.control + offsetof(WtStepControl, skipped));
    s.key0 = mix_host((unsigned)(2 * a.count), (unsigned)a.seed, 0x3C6EF372u);
    s.key1 = mix_host((unsigned)(2 * a.count + 1), (unsigned)a.seed, 0x3C6EF372u);
    return s;
}

template <typename P, int MAX>
cudaError_t step_some(const WtAdamW &a, int from, int n, cudaStream_t st) {
    Table<MAX> tb;
    fill(tb, a, from, n);
    const unsigned chunks = tb.chunk[n];
    if (!chunks) return cudaSuccess;
    const unsigned grid = blocks_for(chunks);
    const Step s = step_of(a);
    if (a.state_bits == 8) adamw8<P, MAX><<<grid, kThreads, 0, st>>>(tb, s);
    else adamw32<P, MAX><<<grid, kThreads, 0, st>>>(tb, s);
    return cudaGetLastError();
}

template <typename P>
cudaError_t step_all(const WtAdamW &a, cudaStream_t st) {
    if (a.n <= kFewTensors) return step_some<P, kFewTensors>(a, 0, a.n, st);
    for (int from = 0; from < a.n; from += kMaxTensors) {
        const int n = a.n - from < kMaxTensors ? a.n - from : kMaxTensors;
        const cudaError_t e = step_some<P, kMaxTensors>(a, from, n, st);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

unsigned norm_grid(const WtGradNorm &a, int from, int n) {
    long long chunks = 0;
    for (int k = from; k < from + n; k++) chunks += chunks_of(a.numel[k]);
    return blocks_for(chunks);
}

template <int MAX>
cudaError_t norm_all(const WtGradNorm &a, cudaStream_t st) {
    unsigned blocks = 0, before = 0;
    for (int from = 0; from < a.n; from += MAX) blocks += norm_grid(a, from, a.n - from < MAX ? a.n - from : MAX);
    for (int from = 0; from < a.n; from += MAX) {
        Table<MAX> tb;
        unsigned chunks = 0;
        tb.n = a.n - from < MAX ? a.n - from : MAX;
        for (int i = 0; i < tb.n; i++) {
            Row &t = tb.row[i];
            t.g = (const void *)a.g[from + i];
            t.numel = a.numel[from + i];
            t.type = a.type[from + i];
            t.wide = aligned(a.g[from + i], t.type == WT_F32 ? 16 : 8);
            tb.chunk[i] = chunks;
            chunks += chunks_of(t.numel);
        }
        tb.chunk[tb.n] = chunks;
        const unsigned grid = norm_grid(a, from, tb.n);
        norm_kernel<MAX><<<grid, kThreads, 0, st>>>(tb, a.partial, blocks, before, a.max_norm, a.control);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
        before += grid;
    }
    return cudaSuccess;
}

}  // namespace

long long grad_norm_partials(int n) { return (long long)kMany * ((n + kMaxTensors - 1) / kMaxTensors); }

cudaError_t launch_adamw(const WtAdamW &a, cudaStream_t st) {
    switch (a.type) {
        case WT_F32: return step_all<float>(a, st);
        case WT_BF16: return step_all<__nv_bfloat16>(a, st);
        default: return step_all<__half>(a, st);
    }
}

cudaError_t launch_grad_norm(const WtGradNorm &a, cudaStream_t st) {
    return a.n <= kFewTensors ? norm_all<kFewTensors>(a, st) : norm_all<kMaxTensors>(a, st);
}

}  // namespace wt
