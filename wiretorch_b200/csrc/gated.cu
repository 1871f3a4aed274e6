// The gated linear recurrence over (B, T, N) and its backward pass:
//
//   decay form:    f_t = a_t,              h_t = f_t h_{t-1} + x_t
//   sigmoid form:  f_t = 1 / (1 + e^-a_t), h_t = f_t h_{t-1} + (1 - f_t) x_t
//
// where starts[b, t] is set the step takes h_{t-1} as 0, and a trial's steps from lengths[b]
// on leave the state as it is and have h = 0. The adjoint runs the other way:
//
//   l_t = dL/dh_t + f_{t+1} l_{t+1}        (dL/dlast in place of the second term at the end)
//   decay:   dx_t = l_t,           da_t = l_t h_{t-1}
//   sigmoid: dx_t = (1 - f_t) l_t, da_t = l_t f_t (1 - f_t) (h_{t-1} - x_t)
//
// Each is a first-order recurrence of some 20 (forward) to 40 (backward) instructions an element
// against 6 to 20 bytes: bound by the bytes of its operands. A thread walks along time with four
// columns of a trial. Where the columns alone do not fill the GPU, time is cut into parts: a step
// is the affine map s -> f s + u, and maps compose, so a first kernel has each thread reduce one
// part of its columns to the part's map s -> A s + H, a small second one joins the maps in order
// into the state that enters each part, and the third walks all parts at once from there. That
// reads two operands twice (from L2 where they fit). One pass, with segments of time held in
// registers and their maps joined over a block or over a cluster's shared memory, reads them
// once, but took 50 instructions an element and waited at its barriers: 32 x 10,000 x 256 bf16
// 0.22 ms forward and 0.46 backward against 0.15 and 0.21, 1 x 131,072 x 64 fp32 0.20 and 0.21
// against 0.05 and 0.06. The product of the decays over a stretch of time has to stay in float's
// range; where growing ones leave it, a state that enters the stretch as 0 is still right.
//
// The backward pass recomputes h inside a segment of kSteps steps from the float state that
// enters it: the forward's own output for float, states it saved on the way for 16-bit types
// (half a byte an element; the output itself, rounded, would put its rounding into da).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "common.cuh"

namespace wt {
namespace {

constexpr int kSteps = WT_GATED_SEGMENT;  // steps of a thread's segment
constexpr int V = 4;                      // columns of a thread
// Threads of a block, where rows allow access to four elements at once and where not: there the SM's
// shared memory holds more of the smaller ones (64 x 500 x 20,000 fp32 1.21 ms with 64 or 128
// threads, 1.18 with 256; 32 x 500 x 20,001 fp32 0.66 with 64 or 128, 0.83 with 256).
__host__ __device__ constexpr int block_of(bool wide) { return wide ? 256 : 128; }
constexpr int kMaxParts = 2048;
// Fewer steps are not cut: 2 x T x 64 fp32 takes 6 us uncut and 8 cut at T = 32, 8 either way at 64,
// 14 and 10 at 128.
constexpr int kLeast = 8 * kSteps;
// Tiles of kSteps steps that are held or on their way, by element size and operands: what keeps the
// memory busy (100 KB an SM on their way) at the most threads.
__host__ __device__ constexpr int stages_of(int size, int ops) { return size == 4 || ops == 3 ? 2 : 3; }
constexpr size_t stage_bytes(int size, int ops, bool wide) { return (size_t)stages_of(size, ops) * ops * kSteps * block_of(wide) * V * size; }

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ void put(float *p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void put(__half *p, float x) { *p = __float2half_rn(x); }

// Four adjacent elements, aligned to their size.
__device__ __forceinline__ void load4(const float *p, float (&x)[V]) {
    const float4 q = *reinterpret_cast<const float4 *>(p);
    x[0] = q.x, x[1] = q.y, x[2] = q.z, x[3] = q.w;
}
__device__ __forceinline__ void load4(const __nv_bfloat16 *p, float (&x)[V]) {
    const uint2 q = *reinterpret_cast<const uint2 *>(p);
    x[0] = __uint_as_float(q.x << 16), x[1] = __uint_as_float(q.x & 0xFFFF0000u);
    x[2] = __uint_as_float(q.y << 16), x[3] = __uint_as_float(q.y & 0xFFFF0000u);
}
__device__ __forceinline__ void load4(const __half *p, float (&x)[V]) {
    const uint2 q = *reinterpret_cast<const uint2 *>(p);
    const float2 u = __half22float2(reinterpret_cast<const __half2 &>(q.x)), v = __half22float2(reinterpret_cast<const __half2 &>(q.y));
    x[0] = u.x, x[1] = u.y, x[2] = v.x, x[3] = v.y;
}
__device__ __forceinline__ void put4(float *p, const float (&x)[V]) {
    *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void put4(__nv_bfloat16 *p, const float (&x)[V]) {
    const __nv_bfloat162 u = __floats2bfloat162_rn(x[0], x[1]), v = __floats2bfloat162_rn(x[2], x[3]);
    *reinterpret_cast<uint2 *>(p) = make_uint2(reinterpret_cast<const unsigned &>(u), reinterpret_cast<const unsigned &>(v));
}
__device__ __forceinline__ void put4(__half *p, const float (&x)[V]) {
    const __half2 u = __floats2half2_rn(x[0], x[1]), v = __floats2half2_rn(x[2], x[3]);
    *reinterpret_cast<uint2 *>(p) = make_uint2(reinterpret_cast<const unsigned &>(u), reinterpret_cast<const unsigned &>(v));
}

// 2^y and 1 / y of the hardware (good to 2^-22 and to a unit in the last place; what would be
// subnormal is 0).
__device__ __forceinline__ float exp2_fast(float y) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
    return r;
}
__device__ __forceinline__ float reciprocal_fast(float y) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
    return r;
}
__device__ __forceinline__ float least(float x, float y) {  // a NaN stays one
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
    return r;
}

// f = 1 / (1 + e^-a) and g = 1 - f = e^-a f, each to its own precision. e^-a = 2^y with
// y = -a log2(e), held below 2^115: there f is under 2^-115 either way, and e^-a f stays 1.
// For float the rounding of y, up to |y| 2^-24, is made good to first order.
template <typename E, bool SIG>
__device__ __forceinline__ void gate(float a, float &f, float &g) {
    if (SIG) {
        constexpr float kLog2e = 1.44269504089f;
        const float y = least(a * -kLog2e, 115.0f);
        float e = exp2_fast(y);
        if (sizeof(E) == 4) {
            constexpr float kLog2eRest = 1.92596299e-08f, kLn2 = 0.69314718056f;  // log2(e) - kLog2e
            const float off = __fmaf_rn(a, -kLog2eRest, __fmaf_rn(a, -kLog2e, -y));
            e = y < 115.0f && y > -115.0f ? __fmaf_rn(e, off * kLn2, e) : e;
        }
        f = reciprocal_fast(1.0f + e);
        g = e * f;
    } else {
        f = a;
        g = 1.0f;
    }
}

// What stands in place of a step past the end: it keeps the state (f = 1) and, with x = 0, adds nothing.
template <typename E, bool SIG>
__device__ __forceinline__ float keeps() {
    return SIG ? __int_as_float(0x7f800000) : 1.0f;
}

// A product of decays: infinity stands for one that overflowed, kTrace of its sign for one that
// underflowed (which is still infinite times an infinite state), 0 for one with a decay of 0 in it, and
// one with a decay that is not finite is not a number.
constexpr float kTrace = 1.401298464e-45f;
__device__ __forceinline__ float product(float A, float a) {
    const float p = A * a;
    if (isnan(p)) return isnan(A) || isnan(a) ? p : 0.0f;
    return p == 0.0f && A != 0.0f && a != 0.0f ? copysignf(kTrace, p) : p;
}

// s -> A s + H. A state of 0 takes no part where a product of growing decays overflowed (a finite one
// takes 1e-45 of itself where a product underflowed).
__device__ __forceinline__ float follow(float A, float H, float s) {
    const float r = __fmaf_rn(A, s, H);
    return isnan(r) && s == 0.0f && !isnan(A) ? H : r;
}

// The threads of a trial's columns, and the columns of a thread: adjacent ones where rows allow
// access to four at once (`wide`), else a warp takes 128 columns, a thread four of them 32 apart, so
// that single accesses of the warp are adjacent.
constexpr int kLanes = 32;
__host__ __device__ inline int threads_of(int N, bool wide) { return wide ? N / V : (N + V * kLanes - 1) / (V * kLanes) * kLanes; }

template <bool WIDE>
struct Columns {
    int n0, N;
    __device__ Columns(int q, int N) : n0(WIDE ? q * V : q / kLanes * (V * kLanes) + q % kLanes), N(N) {}
    __device__ __forceinline__ bool has(int j) const { return WIDE || n0 + j * kLanes < N; }
    __device__ __forceinline__ int tile() const { return n0 & ~(V * kLanes - 1); }  // the warp's first, where not WIDE
    template <typename E>
    __device__ __forceinline__ void get(const E *row, float (&x)[V]) const {
        if (WIDE) {
            load4(row + n0, x);
        } else {
#pragma unroll
            for (int j = 0; j < V; j++)
                if (has(j)) x[j] = to_float(row[n0 + j * kLanes]);
        }
    }
    template <typename E>
    __device__ __forceinline__ void set(E *row, const float (&x)[V]) const {
        if (WIDE) {
            put4(row + n0, x);
        } else {
#pragma unroll
            for (int j = 0; j < V; j++)
                if (has(j)) put(row + n0 + j * kLanes, x[j]);
        }
    }
};

// Operands reach a thread through shared memory: the next tiles' are on their way there
// (asynchronous copies) while one is worked on. Where rows allow access to four elements at once, a
// thread copies into slots of its own what it will read, and no barrier stands between. Copies of
// 16 bytes pass by the L1 cache, whose lines the smaller ones hold until they arrive (with most of
// the L1 given to shared memory that bounds what is on its way: 32 x 500 x 20,000 bf16 took 0.45 ms
// in place of 0.33); so where 16-bit rows allow it, the two threads of adjacent columns share their
// copies, each fetching 16 bytes of one operand for both, and meet (as a warp) around a tile.
template <int BYTES>
__device__ __forceinline__ void copy_async(void *to, const void *from) {
    const unsigned at = (unsigned)__cvta_generic_to_shared(to);
    if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copies_end_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait_all_but() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Where a tile's rows lie in its stage: nothing to know where threads have slots of their own.
template <int OPS, bool WIDE>
struct View {
    int n;  // steps that are there
    template <typename E>
    __device__ View(int n, const E *const (&)[OPS], const long long (&)[OPS], const Columns<WIDE> &) : n(n) {}
};

template <typename E, int OPS, bool WIDE>
struct Stage {
    alignas(16) E slot[OPS][kSteps][block_of(WIDE)][V];
    // Up to kSteps of the operands' `n` steps from their rows `row` on (n is above 0), `other` in
    // place of the ones behind them.
    __device__ __forceinline__ void fetch(int n, const E *(&row)[OPS], const long long (&stride)[OPS], const float (&other)[OPS],
                                          const Columns<WIDE> &col, bool pairs) {
        const int odd = threadIdx.x & 1;
        if (sizeof(E) == 2 && pairs && n >= kSteps) {
            // the even thread fetches the first operand, the odd one the second, and either every other
            // step of the third; each for both
            const int n0 = col.n0 - V * odd, both = threadIdx.x - odd;
            const E *at = (odd ? row[1] : row[0]) + n0;
            const long long step = odd ? stride[1] : stride[0];
#pragma unroll
            for (int k = 0; k < kSteps; k++, at += step) copy_async<16>(slot[odd][k][both], at);
            if (OPS == 3) {
                at = row[OPS - 1] + n0 + odd * stride[OPS - 1];
#pragma unroll
                for (int k = 0; k < kSteps; k += 2, at += 2 * stride[OPS - 1]) copy_async<16>(slot[OPS - 1][k + odd][both], at);
            }
        } else {
            const bool whole = n >= kSteps;
#pragma unroll
            for (int k = 0; k < kSteps; k++)
#pragma unroll
                for (int op = 0; op < OPS; op++) {
                    E *to = slot[op][k][threadIdx.x];
                    if (whole || k < n) {
                        copy_async<V * (int)sizeof(E)>(to, row[op] + col.n0);
                    } else {
                        const float o[V] = {other[op], other[op], other[op], other[op]};
                        put4(to, o);
                    }
                    row[op] += stride[op];
                }
        }
    }
    __device__ __forceinline__ void get(int op, int k, const View<OPS, WIDE> &, float, float (&x)[V]) const {
        load4(slot[op][k][threadIdx.x], x);
    }
};

// Other rows: a warp copies its 128 columns of a row as the aligned pieces of 16 bytes that cover
// them (bytes ahead of the row's share its first piece; the last piece ends where the row ends), and
// each row lies in the stage as far past a multiple of 16 as in memory. 32 x 500 x 20,001 bf16 0.41 ms
// forward, 0.71 backward (4.7 TB/s; the results' rows are written by single accesses), fp32 0.66 and
// 1.32 (5.8 and 5.0); bf16 0.87 and 1.34 with loads of single elements.
template <int OPS>
struct View<OPS, false> {
    int n;
    unsigned at[OPS], step[OPS];
    template <typename E>
    __device__ View(int n, const E *const (&row)[OPS], const long long (&stride)[OPS], const Columns<false> &col) : n(n) {
#pragma unroll
        for (int op = 0; op < OPS; op++) {
            at[op] = (unsigned)((uintptr_t)(row[op] + col.tile()) & 15);
            step[op] = (unsigned)(stride[op] * (long long)sizeof(E)) & 15;
        }
    }
};

template <typename E, int OPS>
struct Stage<E, OPS, false> {
    static constexpr int kPieces = kLanes * V * (int)sizeof(E) / 16;
    alignas(16) unsigned char rows[block_of(false) / kLanes][OPS][kSteps][16 * (kPieces + 1)];
    static __device__ __forceinline__ void piece(unsigned char *to, const E *row, int bytes, int c) {
        const unsigned char *const end = reinterpret_cast<const unsigned char *>(row) + bytes;
        const unsigned char *const from = reinterpret_cast<const unsigned char *>((uintptr_t)row & ~(uintptr_t)15) + 16 * c;
        const int left = (int)min((long long)(end - from), 16LL);
        if (left > 0)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((unsigned)__cvta_generic_to_shared(to + 16 * c)), "l"(from),
                         "r"(left)
                         : "memory");
    }
    __device__ __forceinline__ void fetch(int n, const E *(&row)[OPS], const long long (&stride)[OPS], const float (&)[OPS],
                                          const Columns<false> &col, bool) {
        constexpr int kAtOnce = kLanes / kPieces;  // rows
        const int lane = threadIdx.x % kLanes, w = threadIdx.x / kLanes, c = lane % kPieces, part = lane / kPieces;
        const int bytes = min(V * kLanes, col.N - col.tile()) * (int)sizeof(E);
#pragma unroll
        for (int op = 0; op < OPS; op++) {
            const E *at = row[op] + col.tile() + part * stride[op];
#pragma unroll
            for (int k = 0; k < kSteps; k += kAtOnce, at += kAtOnce * stride[op]) {
                if (k + part < n) {
                    unsigned char *to = rows[w][op][k + part];
                    piece(to, at, bytes, c);
                    if (c == 0) piece(to, at, bytes, kPieces);
                }
            }
        }
    }
    __device__ __forceinline__ void get(int op, int k, const View<OPS, false> &view, float other, float (&x)[V]) const {
        const E *row = reinterpret_cast<const E *>(rows[threadIdx.x / kLanes][op][k] + (view.at[op] + k * view.step[op] & 15));
#pragma unroll
        for (int j = 0; j < V; j++) x[j] = k < view.n ? to_float(row[threadIdx.x % kLanes + j * kLanes]) : other;
    }
};

// The kernels of a call overlap: one may start while the one before it ends, as its room on the
// SMs frees, and waits where it reads what that one wrote.
__device__ __forceinline__ void next_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// The starts among a tile's n steps from t0 on, as bits.
__device__ __forceinline__ unsigned starts_of(const uint8_t *starts, int n) {
    unsigned bits = 0;
#pragma unroll
    for (int k = 0; k < kSteps; k++)
        if (k < n && starts[k]) bits |= 1u << k;
    return bits;
}

// What a thread works on: four columns of a part of a trial's time.
struct Place {
    int b, part, q;
    int lo, hi, len;  // the part's steps, and the trial's
    template <typename Args>
    __device__ Place(const Args &s, int threads, int parts, int part_steps) {
        const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x, per = (long long)threads * parts;
        const long long trial = i >> 32 ? i / per : (long long)((unsigned)i / (unsigned)per);
        const unsigned rest = (unsigned)(i - trial * per);
        part = parts == 1 ? 0 : rest / (unsigned)threads;
        q = rest - part * threads;
        b = trial < s.B ? (int)trial : -1;
        lo = part * part_steps;
        hi = min(lo + part_steps, s.T);
        len = b < 0 || !s.lengths ? s.T : max(0, min(s.lengths[b], s.T));
    }
};

// The maps of the parts: per trial and part a row of A, a row of H and whether a start lies in it
// (what enters the part is dropped). Joined, the row of H is replaced by the state entering the part.
struct Maps {
    float *rows;  // (B, parts, 2, N)
    uint8_t *cut; // (B, parts)
    int parts, part_steps;
    int pairs;  // 16-bit rows allow 16 bytes at once
    __device__ __forceinline__ float *A(int b, int p, int N) const { return rows + ((long long)b * parts + p) * 2 * N; }
    __device__ __forceinline__ float *H(int b, int p, int N) const { return A(b, p, N) + N; }
};

// Each part's map, FORWARD of h' = f h + u, else of adj' = f (adj + dh); `operand` is x or dh. The part is
// walked in its own order from a state of 0, so that H is what the walk behind it would come to: adding each
// step's term times the product of the decays that follow makes 0 times infinity of a term of 0
// where those grow past float's range (and walking against time for it, to begin the next walk with what
// is still in L2, was worth at most 1%: 208 against 210 us of the backward pass of 32 x 10,000 x 256
// bf16). There 57 us, 5.8 TB/s, instructions issued in 60-70% of the cycles.
template <typename E, bool SIG, bool WIDE, bool CUTS, bool FORWARD, typename Args>
__global__ void __launch_bounds__(block_of(WIDE)) maps_kernel(const Args s, const void *operand, long long o_b, long long o_t, const Maps maps) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    auto *stage = reinterpret_cast<Stage<E, 2, WIDE> *>(dynamic);
    constexpr int kHold = stages_of(sizeof(E), 2);
    const Place at(s, threads_of(s.N, WIDE), maps.parts, maps.part_steps);
    constexpr bool kMeet = !WIDE || sizeof(E) == 2;
    const unsigned live = __ballot_sync(kFull, at.b >= 0);
    if (at.b < 0) return;
    const Columns<WIDE> col(at.q, s.N);
    const E *a = static_cast<const E *>(s.a) + at.b * s.a_b, *o = static_cast<const E *>(operand) + at.b * o_b;
    const uint8_t *starts = CUTS ? s.starts + (long long)at.b * s.T : nullptr;
    const int end = min(at.hi, at.len), tiles = end > at.lo ? (end - at.lo + kSteps - 1) / kSteps : 0;
    auto first = [&](int i) { return at.lo + (FORWARD ? i : tiles - 1 - i) * kSteps; };
    auto fetch = [&](int i) {
        const int t0 = first(i);
        const E *row[2] = {a + t0 * s.a_t, o + t0 * o_t};
        const long long stride[2] = {s.a_t, o_t};
        stage[i % kHold].fetch(end - t0, row, stride, {keeps<E, SIG>(), 0.0f}, col, maps.pairs);
    };
    auto view_of = [&](int i) {
        const int t0 = first(i);
        const E *const row[2] = {a + t0 * s.a_t, o + t0 * o_t};
        const long long stride[2] = {s.a_t, o_t};
        return View<2, WIDE>(end - t0, row, stride, col);
    };
#pragma unroll
    for (int i = 0; i < kHold - 1; i++) {
        if (i < tiles) fetch(i);
        copies_end_group();
    }
    next_may_start();
    float A[V] = {1.0f, 1.0f, 1.0f, 1.0f}, H[V] = {}, most[V] = {}, least[V] = {1.0f, 1.0f, 1.0f, 1.0f};
    bool cut = false;  // a start was met: what enters the part is dropped
    const int rounds = kMeet ? __reduce_max_sync(live, tiles) : tiles;
    for (int i = 0; i < rounds; i++) {
        if (kMeet) __syncwarp(live);  // the other thread has read the slots that are filled next
        if (i + kHold - 1 < tiles) fetch(i + kHold - 1);
        copies_end_group();
        copies_wait_all_but<kHold - 1>();
        if (kMeet) __syncwarp(live);  // its copies are here too
        if (kMeet && i >= tiles) continue;
        const auto view = view_of(i);
        const unsigned bits = CUTS ? starts_of(starts + first(i), end - first(i)) : 0;
#pragma unroll
        for (int m = 0; m < kSteps; m++) {
            const int k = FORWARD ? m : kSteps - 1 - m;
            const bool start = CUTS && (bits >> k & 1);
            float f[V], u[V];
            stage[i % kHold].get(0, k, view, keeps<E, SIG>(), f);
            stage[i % kHold].get(1, k, view, 0.0f, u);
#pragma unroll
            for (int j = 0; j < V; j++) {
                float g;
                gate<E, SIG>(f[j], f[j], g);
                if (!SIG) {
                    most[j] = fmaxf(most[j], fabsf(f[j]));
                    least[j] = fminf(least[j], fabsf(f[j]));
                }
                if (FORWARD) {
                    if (SIG) u[j] *= g;
                    H[j] = start ? u[j] : __fmaf_rn(f[j], H[j], u[j]);
                } else {
                    H[j] = start ? 0.0f : f[j] * (H[j] + u[j]);
                }
                A[j] *= f[j];
            }
            cut |= start;
        }
    }
#pragma unroll
    for (int j = 0; j < V; j++) {
        // an infinite decay makes a state of 0 not a number; of finite ones a single 0 makes the product 0,
        // though it may have overflowed; the sigmoid form's are above 0
        if (!SIG && isinf(most[j])) A[j] = CUDART_NAN_F;
        else if (!SIG && least[j] == 0.0f) A[j] = 0.0f;
        else if (A[j] == 0.0f) A[j] = copysignf(kTrace, A[j]);
        if (CUTS && cut) A[j] = 0.0f;
    }
    col.set(maps.A(at.b, at.part, s.N), A);
    col.set(maps.H(at.b, at.part, s.N), H);
    if (CUTS && at.q == 0) maps.cut[(long long)at.b * maps.parts + at.part] = cut;
}

// Joins the maps of a trial's parts into the states that enter them: a block takes COLS columns,
// each of the 32 / COLS x WARPS threads of a column a run of up to RUN parts, held in registers.
// Runs are joined within a warp by shuffles, then over the warps. Latency: 37 parts of 8,192
// columns 6 us, 2,048 parts of 64 columns 10.
template <bool FORWARD, bool CUTS, int COLS, int WARPS, int RUN>
__global__ void __launch_bounds__(32 * WARPS) join_kernel(const Maps maps, const float *state, int N) {
    constexpr int kIn = 32 / COLS, kRuns = kIn * WARPS;
    __shared__ float As[WARPS][COLS], Hs[WARPS][COLS];
    __shared__ int cuts[WARPS];
    const int lane = threadIdx.x % COLS, in = threadIdx.x / COLS % kIn, w = threadIdx.x / 32, b = blockIdx.y;
    const int n = min(blockIdx.x * COLS + lane, N - 1);  // threads past the last column repeat it
    const int each = (maps.parts + kRuns - 1) / kRuns, p0 = (kIn * w + in) * each, mine = min(each, maps.parts - p0);
    const int first = FORWARD ? p0 : maps.parts - 1 - p0;
    const long long stride = (FORWARD ? 2 : -2) * (long long)N;
    float *const rowA = maps.rows + ((long long)b * maps.parts + first) * 2 * N + n, *const rowH = rowA + N;
    const uint8_t *const cut = maps.cut + (long long)b * maps.parts + first;
    float pa[RUN], ph[RUN];
    unsigned c = 0;
    auto all = [&](auto body) {
#pragma unroll
        for (int i = 0; i < RUN; i++)
            if (i < mine) body(i);
    };
    next_may_start();
    const float from = state ? state[(long long)b * N + n] : 0.0f;
    wait_for_last();
    all([&](int i) {
        pa[i] = rowA[i * stride];
        ph[i] = rowH[i * stride];
    });
    if (CUTS) all([&](int i) { c |= (unsigned)(cut[FORWARD ? i : -i] != 0) << i; });
    float A = 1.0f, H = 0.0f;
    int any = 0;
    auto then = [](float &A, float &H, float a, float h, bool cut) {  // (A, H), then (a, h)
        H = cut ? h : follow(a, h, H);
        A = cut ? 0.0f : product(A, a);
    };
    all([&](int i) { then(A, H, pa[i], ph[i], CUTS && (c >> i & 1)); });
    any = c != 0;
#pragma unroll
    for (int o = 1; o < kIn; o <<= 1) {  // inclusive over the warp's runs
        float ua = __shfl_up_sync(kFull, A, COLS * o), uh = __shfl_up_sync(kFull, H, COLS * o);
        const int ucut = CUTS ? __shfl_up_sync(kFull, any, COLS * o) : 0;
        if (in >= o) {
            then(ua, uh, A, H, CUTS && any);
            A = ua;
            H = uh;
            any |= ucut;
        }
    }
    if (in == kIn - 1) {
        As[w][lane] = A;
        Hs[w][lane] = H;
        if (CUTS) cuts[w] = any;
    }
    const float ua = __shfl_up_sync(kFull, A, COLS), uh = __shfl_up_sync(kFull, H, COLS);
    const int ucut = CUTS ? __shfl_up_sync(kFull, any, COLS) : 0;
    __syncthreads();
    float st = from;
    for (int k = 0; k < w; k++) st = CUTS && cuts[k] ? Hs[k][lane] : follow(As[k][lane], Hs[k][lane], st);
    if (in > 0) st = ucut ? uh : follow(ua, uh, st);
    if (blockIdx.x * COLS + lane >= N) return;
    all([&](int i) {
        rowH[i * stride] = st;
        st = CUTS && (c >> i & 1) ? ph[i] : follow(pa[i], ph[i], st);
    });
}

// The walk. 64 x 500 x 20,000 fp32, no parts: 1.17 ms, 6.6 TB/s, what a copy reaches. 32 x 10,000 x
// 256 bf16 in 37 parts: 84 us, 5.9 TB/s of a, x, h and the saved states.
template <typename E, bool SIG, bool WIDE, bool CUTS>
__global__ void __launch_bounds__(block_of(WIDE)) scan_kernel(const WtGatedScan s, const Maps maps) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    auto *stage = reinterpret_cast<Stage<E, 2, WIDE> *>(dynamic);
    constexpr int kHold = stages_of(sizeof(E), 2);
    const Place at(s, threads_of(s.N, WIDE), maps.parts, maps.part_steps);
    constexpr bool kMeet = !WIDE || sizeof(E) == 2;
    const unsigned live = __ballot_sync(kFull, at.b >= 0);
    if (at.b < 0) return;
    const Columns<WIDE> col(at.q, s.N);
    const E *a = static_cast<const E *>(s.a) + at.b * s.a_b, *x = static_cast<const E *>(s.x) + at.b * s.x_b;
    E *h = static_cast<E *>(s.h) + (long long)at.b * s.T * s.N;
    const uint8_t *starts = CUTS ? s.starts + (long long)at.b * s.T : nullptr;
    float *saved = s.saved ? s.saved + (long long)at.b * ((s.T + kSteps - 1) / kSteps) * s.N : nullptr;
    const int end = min(at.hi, at.len), tiles = end > at.lo ? (end - at.lo + kSteps - 1) / kSteps : 0;
    auto fetch = [&](int i) {
        const int t0 = at.lo + i * kSteps;
        const E *row[2] = {a + t0 * s.a_t, x + t0 * s.x_t};
        const long long stride[2] = {s.a_t, s.x_t};
        stage[i % kHold].fetch(end - t0, row, stride, {keeps<E, SIG>(), 0.0f}, col, maps.pairs);
    };
    auto view_of = [&](int i) {
        const int t0 = at.lo + i * kSteps;
        const E *const row[2] = {a + t0 * s.a_t, x + t0 * s.x_t};
        const long long stride[2] = {s.a_t, s.x_t};
        return View<2, WIDE>(end - t0, row, stride, col);
    };
#pragma unroll
    for (int i = 0; i < kHold - 1; i++) {
        if (i < tiles) fetch(i);
        copies_end_group();
    }
    float st[V] = {};
    wait_for_last();
    if (maps.parts > 1) col.get(maps.H(at.b, at.part, s.N), st);
    else if (s.state) col.get(s.state + (long long)at.b * s.N, st);
    const int rounds = kMeet ? __reduce_max_sync(live, tiles) : tiles;
    for (int i = 0; i < rounds; i++) {
        const int t0 = at.lo + i * kSteps;
        if (kMeet) __syncwarp(live);  // the other thread has read the slots that are filled next
        if (i + kHold - 1 < tiles) fetch(i + kHold - 1);
        copies_end_group();
        copies_wait_all_but<kHold - 1>();
        if (kMeet) __syncwarp(live);  // its copies are here too
        if (kMeet && i >= tiles) continue;
        const auto view = view_of(i);
        const unsigned bits = CUTS ? starts_of(starts + t0, end - t0) : 0;
        if (saved) col.set(saved + (long long)(t0 / kSteps) * s.N, st);
        E *ph = h + (long long)t0 * s.N;
#pragma unroll
        for (int k = 0; k < kSteps; k++, ph += s.N) {
            float f[V], u[V];
            stage[i % kHold].get(0, k, view, keeps<E, SIG>(), f);
            stage[i % kHold].get(1, k, view, 0.0f, u);
#pragma unroll
            for (int j = 0; j < V; j++) {
                float g;
                gate<E, SIG>(f[j], f[j], g);
                if (SIG) u[j] *= g;
                st[j] = CUTS && (bits >> k & 1) ? u[j] : __fmaf_rn(f[j], st[j], u[j]);
            }
            if (t0 + k < end) col.set(ph, st);
        }
    }
    const float zero[V] = {};
    for (int t = max(at.lo, at.len); t < at.hi; t++) col.set(h + (long long)t * s.N, zero);
    if (at.part == maps.parts - 1) col.set(s.last + (long long)at.b * s.N, st);
}

// The walk back. 64 x 500 x 20,000 fp32: 2.05 ms, 6.4 TB/s (a, x, dh, da, dx and an eighth of h), with
// decays learnt per column 1.21 ms; 32 x 10,000 x 256 bf16 in 37 parts 135 us, 6.1 TB/s.
template <typename E, bool SIG, bool WIDE, bool CUTS, typename D>
__global__ void __launch_bounds__(block_of(WIDE)) grad_kernel(const WtGatedGrad s, const Maps maps) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    auto *stage = reinterpret_cast<Stage<E, 3, WIDE> *>(dynamic);
    constexpr int kHold = stages_of(sizeof(E), 3);
    const Place at(s, threads_of(s.N, WIDE), maps.parts, maps.part_steps);
    constexpr bool kMeet = !WIDE || sizeof(E) == 2;
    const unsigned live = __ballot_sync(kFull, at.b >= 0);
    if (at.b < 0) return;
    const Columns<WIDE> col(at.q, s.N);
    const E *a = static_cast<const E *>(s.a) + at.b * s.a_b, *x = static_cast<const E *>(s.x) + at.b * s.x_b;
    const E *dh = static_cast<const E *>(s.dh) + at.b * s.dh_b;
    const long long base = (long long)at.b * s.T * s.N;
    E *dx = static_cast<E *>(s.dx) + base;
    D *da = static_cast<D *>(s.da) + (s.reduce ? ((long long)at.b * maps.parts + at.part) * s.N : base);
    const uint8_t *starts = CUTS ? s.starts + (long long)at.b * s.T : nullptr;
    const float *saved = s.saved ? s.saved + (long long)at.b * ((s.T + kSteps - 1) / kSteps) * s.N : nullptr;
    const float *h = static_cast<const float *>(s.h) + base;  // float, where nothing was saved
    const int end = min(at.hi, at.len), tiles = end > at.lo ? (end - at.lo + kSteps - 1) / kSteps : 0;
    auto first = [&](int i) { return at.lo + (tiles - 1 - i) * kSteps; };
    auto fetch = [&](int i) {
        const int t0 = first(i);
        const E *row[3] = {a + t0 * s.a_t, x + t0 * s.x_t, dh + t0 * s.dh_t};
        const long long stride[3] = {s.a_t, s.x_t, s.dh_t};
        stage[i % kHold].fetch(end - t0, row, stride, {keeps<E, SIG>(), 0.0f, 0.0f}, col, maps.pairs);
    };
    auto view_of = [&](int i) {
        const int t0 = first(i);
        const E *const row[3] = {a + t0 * s.a_t, x + t0 * s.x_t, dh + t0 * s.dh_t};
        const long long stride[3] = {s.a_t, s.x_t, s.dh_t};
        return View<3, WIDE>(end - t0, row, stride, col);
    };
    // the state that enters the tile at t0
    auto entering = [&](int t0, float (&st)[V]) {
        const float *row = t0 == 0 ? (s.state ? s.state + (long long)at.b * s.N : nullptr)
                           : saved ? saved + (long long)(t0 / kSteps) * s.N
                                   : h + (long long)(t0 - 1) * s.N;
        if (row) col.get(row, st);
    };
#pragma unroll
    for (int i = 0; i < kHold - 1; i++) {
        if (i < tiles) fetch(i);
        copies_end_group();
    }
    float adj[V] = {}, sum[V] = {}, next[V] = {};
    if (tiles) entering(first(0), next);
    const float zero[V] = {};
    for (int t = max(at.lo, at.len); t < at.hi; t++) {
        col.set(dx + (long long)t * s.N, zero);
        if (!s.reduce) col.set(da + (long long)t * s.N, zero);
    }
    wait_for_last();
    if (maps.parts > 1) col.get(maps.H(at.b, at.part, s.N), adj);
    else if (s.dlast) col.get(s.dlast + (long long)at.b * s.N, adj);
    const int rounds = kMeet ? __reduce_max_sync(live, tiles) : tiles;
    for (int i = 0; i < rounds; i++) {
        const int t0 = first(i);
        if (kMeet) __syncwarp(live);  // the other thread has read the slots that are filled next
        if (i + kHold - 1 < tiles) fetch(i + kHold - 1);
        copies_end_group();
        float prev[V];
#pragma unroll
        for (int j = 0; j < V; j++) {
            prev[j] = next[j];
            next[j] = 0.0f;
        }
        if (i + 1 < tiles) entering(first(i + 1), next);
        copies_wait_all_but<kHold - 1>();
        if (kMeet) __syncwarp(live);  // its copies are here too
        if (kMeet && i >= tiles) continue;
        const auto view = view_of(i);
        const unsigned bits = CUTS ? starts_of(starts + t0, end - t0) : 0;
        float f[kSteps][V], g[SIG ? kSteps : 1][V], w[kSteps][V];  // w: the adjoint's factor of da
#pragma unroll
        for (int k = 0; k < kSteps; k++) {  // h forwards through the tile
            float xk[V];
            stage[i % kHold].get(0, k, view, keeps<E, SIG>(), f[k]);
            stage[i % kHold].get(1, k, view, 0.0f, xk);
#pragma unroll
            for (int j = 0; j < V; j++) {
                float gk;
                gate<E, SIG>(f[k][j], f[k][j], gk);
                if (SIG) g[SIG ? k : 0][j] = gk;
                const float u = SIG ? gk * xk[j] : xk[j];
                const bool start = CUTS && (bits >> k & 1);
                const float from = start ? 0.0f : prev[j];
                prev[j] = start ? u : __fmaf_rn(f[k][j], prev[j], u);
                w[k][j] = SIG ? f[k][j] * gk * (from - xk[j]) : from;
            }
        }
        E *pdx = dx + (long long)(t0 + kSteps - 1) * s.N;
        D *pda = da + (s.reduce ? 0 : (long long)(t0 + kSteps - 1) * s.N);
        const long long back = s.reduce ? 0 : s.N;
#pragma unroll
        for (int k = kSteps - 1; k >= 0; k--, pdx -= s.N, pda -= back) {
            float d[V], gx[V], ga[V];
            stage[i % kHold].get(2, k, view, 0.0f, d);
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float l = adj[j] + d[j];
                gx[j] = SIG ? l * g[SIG ? k : 0][j] : l;
                ga[j] = l * w[k][j];
                adj[j] = CUTS && (bits >> k & 1) ? 0.0f : l * f[k][j];
            }
            if (t0 + k < end) {
                col.set(pdx, gx);
                if (!s.reduce) {
                    col.set(pda, ga);
                } else {
#pragma unroll
                    for (int j = 0; j < V; j++) sum[j] += ga[j];
                }
            }
        }
    }
    if (s.dstate && at.part == 0) col.set(s.dstate + (long long)at.b * s.N, adj);
    if (s.reduce) col.set(da, sum);
}

// One step, a thread per four columns: every operand read and written once, nothing to split.
// 256 x 50,000 bf16: 30 us, 5.9 TB/s; 8 x 1,000 fp32 is a launch.
template <typename E, bool SIG, bool WIDE>
__global__ void __launch_bounds__(256) step_kernel(const WtGatedStep s) {
    const int threads = threads_of(s.N, WIDE);
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long b = i >> 32 ? i / threads : (long long)((unsigned)i / (unsigned)threads);
    if (b >= s.B) return;
    const Columns<WIDE> col((int)(i - b * threads), s.N);
    float a[V] = {}, x[V] = {}, st[V] = {};
    float *state = s.state + b * s.N;
    col.get(static_cast<const E *>(s.a) + b * s.a_b, a);
    col.get(static_cast<const E *>(s.x) + b * s.x_b, x);
    col.get(state, st);
#pragma unroll
    for (int j = 0; j < V; j++) {
        float f, g;
        gate<E, SIG>(a[j], f, g);
        st[j] = __fmaf_rn(f, st[j], SIG ? g * x[j] : x[j]);
    }
    col.set(state, st);
    col.set(static_cast<E *>(s.h) + b * s.N, st);
}

// Steps of a part: whole tiles.
int part_steps_of(int T, int parts) { return ((T + parts - 1) / parts + kSteps - 1) / kSteps * kSteps; }

// The parts time is cut into: as many as the SMs hold threads for at once (a round more would
// leave them waiting for a few last blocks), none shorter than two tiles. By N alone, so that
// neither alignment nor strides move the parts' borders.
int parts_of(int B, int T, int N, int type, bool backward) {
    const bool wide = N % V == 0;
    const int block = block_of(wide);
    const int held = (int)((227 << 10) / (stage_bytes(type == WT_F32 ? 4 : 2, backward ? 3 : 2, wide) * 17 / 16 + 1024));
    const long long columns = (long long)B * threads_of(N, wide);
    const long long full = 148LL * block * (held * block < 1024 ? held : 1024 / block);
    long long parts = full / columns;
    if (parts > T / (2 * kSteps)) parts = T / (2 * kSteps);
    if (parts > kMaxParts) parts = kMaxParts;
    if (parts < 2 || T < kLeast) return 1;
    const int steps = part_steps_of(T, (int)parts);
    return (T + steps - 1) / steps;
}

// Whether rows of a tensor of `size`-byte elements allow access to four at once.
bool fours(const void *p, long long stride_b, long long stride_t, int size) {
    return (uintptr_t)p % (V * size) == 0 && stride_b % V == 0 && stride_t % V == 0;
}

// Whether rows of 16-bit elements allow access to eight at once.
bool eights(const void *p, long long stride_b, long long stride_t) {
    return (uintptr_t)p % 16 == 0 && stride_b % 8 == 0 && stride_t % 8 == 0;
}

// Launches `kernel`. by_l1: its copies pass by the L1 cache, whose room shared memory may take.
// behind: it waits itself for the kernel before it.
template <typename... Params, typename... Args>
cudaError_t launch(void (*kernel)(Params...), dim3 grid, int threads, size_t shared, bool by_l1, bool behind, cudaStream_t st, const Args &...args) {
    if (shared) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                     by_l1 ? cudaSharedmemCarveoutMaxShared : cudaSharedmemCarveoutDefault);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = behind;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <bool FORWARD, int COLS, int WARPS, int RUN>
cudaError_t join_as(const Maps &maps, const float *state, int B, int N, bool cuts, cudaStream_t st) {
    static_assert(32 / COLS * WARPS * RUN <= kMaxParts, "runs");
    const dim3 grid((N + COLS - 1) / COLS, B);
    return launch(cuts ? join_kernel<FORWARD, true, COLS, WARPS, RUN> : join_kernel<FORWARD, false, COLS, WARPS, RUN>, grid, 32 * WARPS, 0,
                  false, true, st, maps, state, N);
}

// The more parts, the fewer columns a block: then the columns are few too, and the SMs many.
template <bool FORWARD>
cudaError_t join(const Maps &maps, const float *state, int B, int N, bool cuts, cudaStream_t st) {
    if (maps.parts <= 64) return join_as<FORWARD, 8, 8, 2>(maps, state, B, N, cuts, st);
    if (maps.parts <= 512) return join_as<FORWARD, 4, 16, 4>(maps, state, B, N, cuts, st);
    return join_as<FORWARD, 2, 32, 4>(maps, state, B, N, cuts, st);
}

Maps maps_of(void *scratch, int B, int T, int N, int type, bool backward, bool pairs) {
    Maps m{};
    m.parts = parts_of(B, T, N, type, backward);
    m.part_steps = part_steps_of(T, m.parts);
    m.rows = static_cast<float *>(scratch);
    m.cut = reinterpret_cast<uint8_t *>(m.rows + (size_t)B * m.parts * 2 * N);
    m.pairs = pairs;
    return m;
}

template <typename E, bool SIG, bool WIDE, bool CUTS>
cudaError_t scan_as(const WtGatedScan &s, cudaStream_t st) {
    const Maps maps = maps_of(s.scratch, s.B, s.T, s.N, s.type, false,
                              s.N % 8 == 0 && eights(s.a, s.a_b, s.a_t) && eights(s.x, s.x_b, s.x_t));
    const bool by_l1 = !WIDE || sizeof(E) == 4 || maps.pairs;
    const dim3 grid((unsigned)(((long long)s.B * maps.parts * threads_of(s.N, WIDE) + block_of(WIDE) - 1) / block_of(WIDE)));
    const size_t shared = stages_of(sizeof(E), 2) * sizeof(Stage<E, 2, WIDE>);
    if (maps.parts > 1) {
        cudaError_t e = launch(maps_kernel<E, SIG, WIDE, CUTS, true, WtGatedScan>, grid, block_of(WIDE), shared, by_l1, false, st, s, s.x, s.x_b, s.x_t, maps);
        if (e == cudaSuccess) e = join<true>(maps, s.state, s.B, s.N, CUTS, st);
        if (e != cudaSuccess) return e;
    }
    return launch(scan_kernel<E, SIG, WIDE, CUTS>, grid, block_of(WIDE), shared, by_l1, maps.parts > 1, st, s, maps);
}

template <typename E, bool SIG, bool WIDE, bool CUTS, typename D>
cudaError_t grad_as(const WtGatedGrad &s, cudaStream_t st) {
    const Maps maps = maps_of(s.scratch, s.B, s.T, s.N, s.type, true,
                              s.N % 8 == 0 && eights(s.a, s.a_b, s.a_t) && eights(s.x, s.x_b, s.x_t) && eights(s.dh, s.dh_b, s.dh_t));
    const bool by_l1 = !WIDE || sizeof(E) == 4 || maps.pairs;
    const dim3 grid((unsigned)(((long long)s.B * maps.parts * threads_of(s.N, WIDE) + block_of(WIDE) - 1) / block_of(WIDE)));
    if (maps.parts > 1) {
        cudaError_t e = launch(maps_kernel<E, SIG, WIDE, CUTS, false, WtGatedGrad>, grid, block_of(WIDE), stages_of(sizeof(E), 2) * sizeof(Stage<E, 2, WIDE>), by_l1, false, st,
                               s, s.dh, s.dh_b, s.dh_t, maps);
        if (e == cudaSuccess) e = join<false>(maps, s.dlast, s.B, s.N, CUTS, st);
        if (e != cudaSuccess) return e;
    }
    return launch(grad_kernel<E, SIG, WIDE, CUTS, D>, grid, block_of(WIDE), stages_of(sizeof(E), 3) * sizeof(Stage<E, 3, WIDE>), by_l1, maps.parts > 1, st, s, maps);
}

template <typename E, bool SIG>
cudaError_t scan_typed(const WtGatedScan &s, cudaStream_t st) {
    const int z = sizeof(E);
    const bool wide = s.N % V == 0 && fours(s.a, s.a_b, s.a_t, z) && fours(s.x, s.x_b, s.x_t, z) && fours(s.h, 0, 0, z) &&
                      fours(s.state, 0, 0, 4) && fours(s.last, 0, 0, 4) && fours(s.saved, 0, 0, 4) && fours(s.scratch, 0, 0, 4);
    if (s.starts) return wide ? scan_as<E, SIG, true, true>(s, st) : scan_as<E, SIG, false, true>(s, st);
    return wide ? scan_as<E, SIG, true, false>(s, st) : scan_as<E, SIG, false, false>(s, st);
}

template <typename E, bool SIG, typename D>
cudaError_t grad_typed(const WtGatedGrad &s, cudaStream_t st) {
    const int z = sizeof(E);
    const bool wide = s.N % V == 0 && fours(s.a, s.a_b, s.a_t, z) && fours(s.x, s.x_b, s.x_t, z) &&
                      fours(s.dh, s.dh_b, s.dh_t, z) && fours(s.dx, 0, 0, z) && fours(s.da, 0, 0, sizeof(D)) &&
                      fours(s.state, 0, 0, 4) && fours(s.h, 0, 0, 4) && fours(s.saved, 0, 0, 4) && fours(s.dlast, 0, 0, 4) &&
                      fours(s.dstate, 0, 0, 4) && fours(s.scratch, 0, 0, 4);
    if (s.starts) return wide ? grad_as<E, SIG, true, true, D>(s, st) : grad_as<E, SIG, false, true, D>(s, st);
    return wide ? grad_as<E, SIG, true, false, D>(s, st) : grad_as<E, SIG, false, false, D>(s, st);
}

template <typename E>
cudaError_t grad_of(const WtGatedGrad &s, cudaStream_t st) {
    const bool sig = s.form == WT_GATED_SIGMOID;
    if (s.da_type == WT_F32) return sig ? grad_typed<E, true, float>(s, st) : grad_typed<E, false, float>(s, st);
    return sig ? grad_typed<E, true, E>(s, st) : grad_typed<E, false, E>(s, st);
}

}  // namespace

int gated_parts(int B, int T, int N, int type, bool backward) { return parts_of(B, T, N, type, backward); }

cudaError_t launch_gated_scan(const WtGatedScan &s, cudaStream_t st) {
    const bool sig = s.form == WT_GATED_SIGMOID;
    switch (s.type) {
        case WT_F32: return sig ? scan_typed<float, true>(s, st) : scan_typed<float, false>(s, st);
        case WT_BF16: return sig ? scan_typed<__nv_bfloat16, true>(s, st) : scan_typed<__nv_bfloat16, false>(s, st);
        default: return sig ? scan_typed<__half, true>(s, st) : scan_typed<__half, false>(s, st);
    }
}

cudaError_t launch_gated_grad(const WtGatedGrad &s, cudaStream_t st) {
    switch (s.type) {
        case WT_F32: return grad_of<float>(s, st);
        case WT_BF16: return grad_of<__nv_bfloat16>(s, st);
        default: return grad_of<__half>(s, st);
    }
}

template <typename E>
static cudaError_t step_of(const WtGatedStep &s, cudaStream_t st) {
    const int z = sizeof(E);
    const bool wide = s.N % V == 0 && fours(s.a, s.a_b, 0, z) && fours(s.x, s.x_b, 0, z) && fours(s.h, 0, 0, z) && fours(s.state, 0, 0, 4);
    const dim3 grid((unsigned)(((long long)s.B * threads_of(s.N, wide) + 255) / 256));
    if (s.form == WT_GATED_SIGMOID)
        return launch(wide ? step_kernel<E, true, true> : step_kernel<E, true, false>, grid, 256, 0, false, false, st, s);
    return launch(wide ? step_kernel<E, false, true> : step_kernel<E, false, false>, grid, 256, 0, false, false, st, s);
}

cudaError_t launch_gated_step(const WtGatedStep &s, cudaStream_t st) {
    switch (s.type) {
        case WT_F32: return step_of<float>(s, st);
        case WT_BF16: return step_of<__nv_bfloat16>(s, st);
        default: return step_of<__half>(s, st);
    }
}

}  // namespace wt
