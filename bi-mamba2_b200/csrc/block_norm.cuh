// The norms before and after a block in one pass over a row (rms(t) = t rstd(t), rstd(t) = 1 / sqrt(mean(t^2) + eps)):
//     n = rms(x) w2,   m = scale act(gate),   r = residual + m n,   u = rms(r) w1
// and its gradients (t = u's gradient times w1, r^ = rms(r), x^ = rms(x)):
//     dr' = dr + rstd(r) (t - r^ mean(t r^)),   dresidual = dr',   dn = dr' m,   dw1 = sum_rows du r^,   dw2 = sum_rows dn x^,
//     dx = rstd(x) (dn w2 - x^ mean(dn w2 x^)),   dscale = sum_rows dr' act(gate) n,   dgate = dr' scale n act'(gate)
// Bound by the rows' bytes: each tensor is read or written once, everything between stays in registers.  A row has
// width / 8 threads with eight channels each - neighbouring ones (16-byte accesses, or by pairs where the width is even and no more), or
// where width or addresses do not allow that, ones a stride apart - and a block walks rows with the weights in registers.  Where neighbours are a thread's, its pieces of the
// next rows come by asynchronous copies into shared memory of its own, several rows ahead: held in registers, one row ahead, they
// left two blocks an SM waiting.  Above 4096 channels a row of the backward pass is two blocks' of a cluster: one block of 1024
// threads left a thread 64 registers, too few (1445 us for 950, 16004 gated rows of 8192; the forward pass, which fits, loses by the
// meetings of a pair, 472 us for 365).  Arithmetic is on pairs of channels (two multiply-adds an instruction).  r is formed
// again in the backward pass, from what the forward pass read, so that no rounding of it enters.  Sums over rows: in registers over a
// block's rows - act, w2 and scale are factors of them that wait until the end, so that dw2, dscale and the gradient of a shared gate row
// come from one sum of dr' x^ (act) - then over the blocks in a second kernel, always in one order.
// Measured: 65536 gated bf16 rows of 1024, forward 123 us (0.67 GB, 5.4 TB/s), backward 183 (1.07 GB, 5.9 TB/s) and 9 for the sums.
#pragma once
#include <type_traits>

#include "common.cuh"
#include "vec.cuh"

namespace bissd {
namespace bnorm {

using vec::add2;
using vec::f2;
using vec::fma2;
using vec::mul2;
using vec::pack;
using vec::unpack;

constexpr int kCh = 8, kPairs = kCh / 2;                         // channels a thread
constexpr int kMaxWidth = 8192;

struct Params {
    int rows, gate_rows;                                         // gate_rows: rows of x to a row of the gate, 0 where each has its own
    int D, threads_row, w_dtype, act, blocks;                    // blocks: of an entry
    float scale, eps;
    int sx, sres, sgate, sdr, sdu;                               // row strides
    const void *x, *res, *gate, *scale_v, *w2, *w1;
    void *r, *u;
    float *rstd;                                                 // [2][rows]: of x, of r
    const void *dr, *du;
    void *dx, *dres, *dgate;
    float *part;                                                 // [blocks][4][D]: dw1, dw2, dscale, dgate of a shared row
};

// Channel e of thread t of a row.  VEC: 8 where a thread's eight channels are neighbours that 16-byte accesses fit, 2 where pairs of them
// are what lies aligned, 0 where they lie a stride apart, single (2790 rows of 4236, forward: 45 us by pairs, 89 single).
template <int VEC> __device__ __forceinline__ int channel(int t, int tr, int e) { return VEC ? t * kCh + e : t + e * tr; }

// A thread's eight channels of one tensor, and how a row's get into registers.
template <class T, int VEC> struct Column {
    static constexpr int kCells = VEC ? kCh * (int)sizeof(T) / 16 : 0;   // of 16 bytes, that a row takes in shared memory
    static constexpr int kPiece = VEC == 8 ? 16 : 2 * (int)sizeof(T), kPieces = kCells * 16 / kPiece;   // how it comes there
    int slot;                                                    // first piece's place in the ring's stage, in bytes
    __device__ __forceinline__ void start(int threads, int *bytes) {
        slot = *bytes;
        *bytes += kCells * threads * 16;
    }
    // A row on its way: zeros where there is none, or no such channels.  Addresses are made anew from the parameters, a multiply-add each:
    // kept and advanced they cost registers that the backward kernel does not have (16 us of 285, 65536 rows of 1024).
    __device__ __forceinline__ void copy(const void *p, int row, int stride, int t, int D, uint32_t stage, int threads, bool in) const {
        if constexpr (VEC == 8) {
            const T *at = static_cast<const T *>(p) + ((long long)row * stride + t * kCh);
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(stage + slot + i * threads * 16),
                             "l"(reinterpret_cast<const uint4 *>(at) + i), "r"(in ? 16 : 0) : "memory");
        } else if constexpr (VEC == 2) {
            const T *at = static_cast<const T *>(p) + ((long long)row * stride + t * kCh);
#pragma unroll
            for (int i = 0; i < kPieces; ++i)                    // a pair of channels
                asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(stage + slot + i * kPiece / 16 * threads * 16 + i * kPiece % 16),
                             "l"(at + 2 * i), "n"(kPiece), "r"(in && t * kCh + 2 * i < D ? kPiece : 0) : "memory");
        }
    }
    __device__ __forceinline__ void get(const void *p, int at_row, int stride, const uint8_t *stage, int threads, int t, int tr, int D,
                                        bool valid, f2 (&v)[kPairs]) const {
        vec::Row<T, kPairs> row;
        if constexpr (VEC > 0) {
#pragma unroll
            for (int i = 0; i < kCells; ++i) {
                const uint4 q = *reinterpret_cast<const uint4 *>(stage + slot + i * threads * 16);
                if constexpr (sizeof(T) == 4) {
                    row.v[2 * i] = make_float2(__uint_as_float(q.x), __uint_as_float(q.y));
                    row.v[2 * i + 1] = make_float2(__uint_as_float(q.z), __uint_as_float(q.w));
                } else {
                    row.v[0] = q.x; row.v[1] = q.y; row.v[2] = q.z; row.v[3] = q.w;
                }
            }
#pragma unroll
            for (int i = 0; i < kPairs; ++i) v[i] = vec::widen<T>(row.v[i]);
        } else {
            const T *at = static_cast<const T *>(p) + (long long)at_row * stride;
            float e[kCh];
#pragma unroll
            for (int i = 0; i < kCh; ++i) e[i] = valid && t + i * tr < D ? to_f<T>(at[t + i * tr]) : 0.f;
#pragma unroll
            for (int i = 0; i < kPairs; ++i) v[i] = pack(e[2 * i], e[2 * i + 1]);
        }
    }
};
template <class T, int VEC>
__device__ __forceinline__ void put(void *p, long long row, int t, int tr, int D, const f2 (&v)[kPairs]) {
    T *base = static_cast<T *>(p) + row * D;
    if constexpr (VEC == 2) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i)
            if (t * kCh + 2 * i < D) *reinterpret_cast<typename vec::Pair<T>::raw *>(base + t * kCh + 2 * i) = vec::narrow<T>(v[i]);
    } else if constexpr (VEC == 8) {
        if (t * kCh >= D) return;
        vec::Row<T, kPairs> o;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) o.v[i] = vec::narrow<T>(v[i]);
        vec::store_row<T, kPairs>(base + t * kCh, o);
    } else {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            float a, b;
            unpack(v[i], a, b);
            if (t + 2 * i * tr < D) base[t + 2 * i * tr] = from_f<T>(a);
            if (t + (2 * i + 1) * tr < D) base[t + (2 * i + 1) * tr] = from_f<T>(b);
        }
    }
}
template <int VEC> __device__ __forceinline__ void weights(const void *p, int dtype, float none, int t, int tr, int D, f2 (&w)[kPairs]) {
    float e[kCh];
#pragma unroll
    for (int i = 0; i < kCh; ++i) {
        const int c = channel<VEC>(t, tr, i);
        e[i] = p ? (c < D ? ld_any(p, dtype, c) : 0.f) : none;
    }
#pragma unroll
    for (int i = 0; i < kPairs; ++i) w[i] = pack(e[2 * i], e[2 * i + 1]);
}
__device__ __forceinline__ float both(f2 v) {
    float a, b;
    unpack(v, a, b);
    return a + b;
}

// Sum over the threads of a row; every thread of the block calls.  The two buffers take turns: who writes one again has met the
// others in the call between.  A row of at most eight warps has eight places, zeros behind its warps' sums, so that two wide reads
// fetch them all: read one by one, their
// place found by a division, they cost 339 us instead of 310 (65536 rows of 1024, gated, forward and backward).
// A row of two blocks: both write all sums, and meet.
template <bool PAIR> struct RowSums {
    float at[2][32];
    __device__ __forceinline__ static void meet() {              // the cluster's blocks; whole warps call
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    __device__ __forceinline__ void start() {
        if (threadIdx.x < 64) at[threadIdx.x >> 5][threadIdx.x & 31] = 0.f;
        if (PAIR)
            meet();                                              // the other block has begun
        else
            __syncthreads();
    }
    __device__ __forceinline__ float operator()(float v, int &turn, int tr, int row) {   // row: of the block's
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (!PAIR && tr == 32) return v;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per = tr >> 5;
        float *buf = at[turn];
        turn ^= 1;
        if (!PAIR && per <= 8) {
            if (lane == 0) buf[row * 8 + warp - row * per] = v;
            __syncthreads();
            const float4 *w = reinterpret_cast<const float4 *>(buf + row * 8);
            const float4 a = w[0], b = w[1];
            return ((((((a.x + a.y) + a.z) + a.w) + b.x) + b.y) + b.z) + b.w;
        }
        if (PAIR) {                                              // lanes 0 and 1: to either block
            if (lane < 2) {
                uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(buf + (blockIdx.x & 1) * (per >> 1) + warp));
                asm volatile("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(to) : "r"(lane));
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(v) : "memory");
            }
            meet();
        } else {                                                 // one row a block
            if (lane == 0) buf[warp] = v;
            __syncthreads();
        }
        float s = lane < per ? buf[lane] : 0.f;                  // a lane for each warp
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        return s;
    }
};

// act of a gate and its slope.
__device__ __forceinline__ void activation(int act, f2 (&a)[kPairs], f2 (&slope)[kPairs]) {
    if (act == BISSD_GATE_NONE) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) slope[i] = pack(1.f, 1.f);
    } else if (act == BISSD_GATE_SIGMOID) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            a[i] = vec::sigmoid2(a[i]);
            slope[i] = fma2(mul2(a[i], pack(-1.f, -1.f)), a[i], a[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            const f2 s = vec::sigmoid2(a[i]);
            slope[i] = vec::silu_slope2(a[i], s);
            a[i] = mul2(a[i], s);
        }
    }
}

// Rows that a thread copies ahead: as many as leave an SM's blocks their shared memory.
template <class T, int THREADS, int PER_SM> struct Ahead {
    static constexpr int rows = THREADS <= 256 ? (sizeof(T) == 4 ? 2 : 4) : THREADS <= 512 ? (PER_SM == 1 && sizeof(T) == 2 ? 3 : 2) : sizeof(T) == 2 ? 2 : 1;
};

// What both kernels walk: rows first + i of an entry (the rows that share a gate row, or all), i = blk per + grp, + step, ...  A row
// behind the last is one of zeros, of which nothing is kept.  PAIR: a row is a cluster's of two blocks.
struct Walk {
    int tr, per, grp, t, D, blk, entry, n, first, step;
    __device__ __forceinline__ Walk(const Params &a, bool pair) {
        const int x = pair ? blockIdx.x >> 1 : blockIdx.x;
        tr = a.threads_row; per = pair ? 1 : blockDim.x / tr; grp = pair ? 0 : threadIdx.x / tr;
        t = pair ? (blockIdx.x & 1) * blockDim.x + threadIdx.x : threadIdx.x % tr; D = a.D;
        blk = x % a.blocks; entry = x / a.blocks;
        n = a.gate && a.gate_rows > 0 ? a.gate_rows : a.rows;
        first = entry * n;
        step = a.blocks * per;
    }
};

template <class T, class R, int VEC, bool PAIR, int THREADS, int PER_SM>
__global__ void __launch_bounds__(THREADS, PER_SM) block_norm_fwd(Params a) {
    pdl_begin();
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ __align__(16) RowSums<PAIR> row_sum;
    row_sum.start();
    const Walk k(a, PAIR);
    const int t = k.t, tr = k.tr, D = k.D, threads = blockDim.x;
    const bool full = a.gate && a.gate_rows == 0, in = t * kCh < D;
    f2 mw[kPairs], w1[kPairs], scw[kPairs];                      // scale act w2; scale w2
    {
        f2 w2[kPairs], sc[kPairs];
        weights<VEC>(a.w2, a.w_dtype, 1.f, t, tr, D, w2);
        weights<VEC>(a.w1, a.w_dtype, 0.f, t, tr, D, w1);
        weights<VEC>(a.scale_v, a.w_dtype, a.scale, t, tr, D, sc);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) mw[i] = scw[i] = mul2(sc[i], w2[i]);
    }
    constexpr int kAhead = Ahead<T, THREADS, PER_SM>::rows;
    const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(dyn)) + threadIdx.x * 16;
    int bytes = 0, turn = 0, at = 0;                             // of a stage of the ring; the stage in turn, in bytes
    int i = k.blk * k.per + k.grp, ahead = i;
    Column<T, VEC> cx, cg;
    Column<R, VEC> cr;
    cx.start(threads, &bytes);
    cr.start(threads, &bytes);
    if (full) cg.start(threads, &bytes);
    auto copy = [&](int stage) {
        const bool some = in && ahead < k.n;
        const int to = k.first + ahead;
        cx.copy(a.x, to, a.sx, t, D, ring + stage, threads, some);
        cr.copy(a.res, to, a.sres, t, D, ring + stage, threads, some);
        if (full) cg.copy(a.gate, to, a.sgate, t, D, ring + stage, threads, some);
        asm volatile("cp.async.commit_group;" ::: "memory");
        ahead += k.step;
    };
    if (a.gate && !full) {
        f2 slope[kPairs];
        const T *p = static_cast<const T *>(a.gate) + (long long)k.entry * a.sgate;
        float e[kCh];
#pragma unroll
        for (int j = 0; j < kCh; ++j) e[j] = channel<VEC>(t, tr, j) < D ? to_f<T>(p[channel<VEC>(t, tr, j)]) : 0.f;
        f2 g[kPairs];
#pragma unroll
        for (int j = 0; j < kPairs; ++j) g[j] = pack(e[2 * j], e[2 * j + 1]);
        activation(a.act, g, slope);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) mw[j] = mul2(g[j], scw[j]);
    }
    if (VEC)
        for (int s = 0; s < kAhead; ++s) copy(s * bytes);
    const float inv = 1.f / D;
    for (int base = k.blk * k.per; base < k.n; base += k.step, i += k.step) {
        const bool valid = i < k.n;
        const int row = k.first + i;
        f2 x[kPairs], r[kPairs];
        const uint8_t *stage = dyn + at + threadIdx.x * 16;
        if (VEC) asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");   // the oldest row has landed
        cx.get(a.x, row, a.sx, stage, threads, t, tr, D, valid, x);
        cr.get(a.res, row, a.sres, stage, threads, t, tr, D, valid, r);
        if (full) {
            f2 g[kPairs], slope[kPairs];
            cg.get(a.gate, row, a.sgate, stage, threads, t, tr, D, valid, g);
            activation(a.act, g, slope);
#pragma unroll
            for (int j = 0; j < kPairs; ++j) mw[j] = mul2(g[j], scw[j]);
        }
        if (VEC) {                                               // its values are in registers: the row kAhead on takes its place
            copy(at);
            at = at + bytes == kAhead * bytes ? 0 : at + bytes;
        }
        float rx = 1.f;
        if (a.w2) {
            f2 q = mul2(x[0], x[0]);
#pragma unroll
            for (int j = 1; j < kPairs; ++j) q = fma2(x[j], x[j], q);
            rx = rsqrtf(row_sum(both(q), turn, tr, k.grp) * inv + a.eps);
            if (a.rstd && t == 0 && valid) a.rstd[row] = rx;
        }
        const f2 rx2 = pack(rx, rx);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) r[j] = fma2(mul2(x[j], rx2), mw[j], r[j]);
        if (valid) put<R, VEC>(a.r, row, t, tr, D, r);
        if (a.u) {
            f2 q = mul2(r[0], r[0]);
#pragma unroll
            for (int j = 1; j < kPairs; ++j) q = fma2(r[j], r[j], q);
            const float rr = rsqrtf(row_sum(both(q), turn, tr, k.grp) * inv + a.eps);
            if (a.rstd && t == 0 && valid) a.rstd[a.rows + row] = rr;
            const f2 rr2 = pack(rr, rr);
#pragma unroll
            for (int j = 0; j < kPairs; ++j) r[j] = mul2(mul2(r[j], rr2), w1[j]);
            if (valid) put<T, VEC>(a.u, row, t, tr, D, r);
        }
    }
    if (VEC) asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <class T, class R, int VEC, bool PAIR, int THREADS, int PER_SM>
__global__ void __launch_bounds__(THREADS, PER_SM) block_norm_bwd(Params a) {
    pdl_begin();
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ __align__(16) RowSums<PAIR> row_sum;
    row_sum.start();
    const Walk k(a, PAIR);
    const int t = k.t, tr = k.tr, D = k.D, threads = blockDim.x;
    const bool full = a.gate && a.gate_rows == 0, in = t * kCh < D;
    f2 w1[kPairs], scw[kPairs], act[kPairs], slope[kPairs], d1[kPairs], d2[kPairs];   // scw: scale w2; d2: sums of dr' x^ (act)
    {
        f2 w2[kPairs], sc[kPairs];
        weights<VEC>(a.w2, a.w_dtype, 1.f, t, tr, D, w2);
        weights<VEC>(a.w1, a.w_dtype, 0.f, t, tr, D, w1);
        weights<VEC>(a.scale_v, a.w_dtype, a.scale, t, tr, D, sc);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
            scw[i] = mul2(sc[i], w2[i]);
            act[i] = slope[i] = pack(1.f, 1.f);
            d1[i] = d2[i] = pack(0.f, 0.f);
        }
    }
    if (a.gate && !full) {
        const T *p = static_cast<const T *>(a.gate) + (long long)k.entry * a.sgate;
        float e[kCh];
#pragma unroll
        for (int j = 0; j < kCh; ++j) e[j] = channel<VEC>(t, tr, j) < D ? to_f<T>(p[channel<VEC>(t, tr, j)]) : 0.f;
#pragma unroll
        for (int j = 0; j < kPairs; ++j) act[j] = pack(e[2 * j], e[2 * j + 1]);
        activation(a.act, act, slope);
    }
    constexpr int kAhead = Ahead<T, THREADS, PER_SM>::rows;
    const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(dyn)) + threadIdx.x * 16;
    int bytes = 0, turn = 0, at = 0;
    int i = k.blk * k.per + k.grp, ahead = i;
    Column<T, VEC> cx, cg, cu;
    Column<R, VEC> cr, cd;
    cx.start(threads, &bytes);
    cr.start(threads, &bytes);
    if (full) cg.start(threads, &bytes);
    if (a.du) cu.start(threads, &bytes);
    if (a.dr) cd.start(threads, &bytes);
    auto copy = [&](int stage) {
        const bool some = in && ahead < k.n;
        const int to = k.first + ahead;
        cx.copy(a.x, to, a.sx, t, D, ring + stage, threads, some);
        cr.copy(a.res, to, a.sres, t, D, ring + stage, threads, some);
        if (full) cg.copy(a.gate, to, a.sgate, t, D, ring + stage, threads, some);
        if (a.du) cu.copy(a.du, to, a.sdu, t, D, ring + stage, threads, some);
        if (a.dr) cd.copy(a.dr, to, a.sdr, t, D, ring + stage, threads, some);
        asm volatile("cp.async.commit_group;" ::: "memory");
        ahead += k.step;
    };
    if (VEC)
        for (int s = 0; s < kAhead; ++s) copy(s * bytes);
    const float inv = 1.f / D;
    float rx_next, rr_next;                                      // of the next row: loaded when needed they made every row wait (265 us for 211)
    auto rstd = [&](int i) {
        const bool valid = i < k.n;
        rx_next = !a.w2 ? 1.f : valid ? a.rstd[k.first + i] : 0.f;
        rr_next = a.du && valid ? a.rstd[a.rows + k.first + i] : 0.f;
    };
    rstd(i);
    for (int base = k.blk * k.per; base < k.n; base += k.step, i += k.step) {
        const bool valid = i < k.n;
        const int row = k.first + i;
        const float rx = rx_next, rr = rr_next;
        rstd(i + k.step);
        const uint8_t *stage = dyn + at + threadIdx.x * 16;
        f2 xh[kPairs], r[kPairs], dr[kPairs], du[kPairs];
        if (VEC) asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");   // the oldest row has landed
        cx.get(a.x, row, a.sx, stage, threads, t, tr, D, valid, xh);
        cr.get(a.res, row, a.sres, stage, threads, t, tr, D, valid, r);
        if (full) cg.get(a.gate, row, a.sgate, stage, threads, t, tr, D, valid, act);
        if (a.du) cu.get(a.du, row, a.sdu, stage, threads, t, tr, D, valid, du);
        if (a.dr) cd.get(a.dr, row, a.sdr, stage, threads, t, tr, D, valid, dr);
        if (VEC) {
            copy(at);
            at = at + bytes == kAhead * bytes ? 0 : at + bytes;
        }
        if (full) activation(a.act, act, slope);
        const f2 rx2 = pack(rx, rx), rr2 = pack(rr, rr);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
            xh[j] = mul2(xh[j], rx2);
            if (!a.dr) dr[j] = pack(0.f, 0.f);
        }
        if (a.du) {
            f2 q = pack(0.f, 0.f);
#pragma unroll
            for (int j = 0; j < kPairs; ++j) {
                r[j] = mul2(fma2(mul2(act[j], scw[j]), xh[j], r[j]), rr2);   // rms(r)
                d1[j] = fma2(du[j], r[j], d1[j]);
                du[j] = mul2(du[j], w1[j]);
                q = fma2(du[j], r[j], q);
            }
            const float c = -rr * (row_sum(both(q), turn, tr, k.grp) * inv);
            const f2 c2 = pack(c, c);
#pragma unroll
            for (int j = 0; j < kPairs; ++j) dr[j] = fma2(r[j], c2, fma2(du[j], rr2, dr[j]));
        }
        if (valid && a.dres) put<R, VEC>(a.dres, row, t, tr, D, dr);
        f2 q = pack(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
            const f2 z = mul2(dr[j], xh[j]);
            d2[j] = full ? fma2(z, act[j], d2[j]) : add2(z, d2[j]);
            du[j] = mul2(mul2(z, scw[j]), slope[j]);             // the gate's
            dr[j] = mul2(dr[j], mul2(act[j], scw[j]));
            q = fma2(dr[j], xh[j], q);
        }
        if (full && a.dgate && valid) put<T, VEC>(a.dgate, row, t, tr, D, du);
        if (a.dx) {
            if (a.w2) {
                const float c = -rx * (row_sum(both(q), turn, tr, k.grp) * inv);
                const f2 c2 = pack(c, c);
#pragma unroll
                for (int j = 0; j < kPairs; ++j) dr[j] = fma2(xh[j], c2, mul2(dr[j], rx2));
            }
            if (valid) put<T, VEC>(a.dx, row, t, tr, D, dr);
        }
    }
    if (VEC) asm volatile("cp.async.wait_group 0;" ::: "memory");
    // rows side by side in this block added up, then one partial row a block
    float *sums = reinterpret_cast<float *>(dyn);
    const long long part = (long long)(PAIR ? blockIdx.x >> 1 : blockIdx.x) * 4 * D;
#pragma unroll
    for (int what = 0; what < 2; ++what) {
        f2(&v)[kPairs] = what ? d2 : d1;
        __syncthreads();                                         // the ring, or the sums before, are no longer read
        if (k.grp > 0) {
#pragma unroll
            for (int j = 0; j < kPairs; ++j) unpack(v[j], sums[((k.grp - 1) * tr + t) * kCh + 2 * j], sums[((k.grp - 1) * tr + t) * kCh + 2 * j + 1]);
        }
        __syncthreads();
        if (k.grp > 0) continue;
        float s[kCh], ac[kCh], sl[kCh], sw[kCh];
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
            unpack(v[j], s[2 * j], s[2 * j + 1]);
            unpack(act[j], ac[2 * j], ac[2 * j + 1]);
            unpack(slope[j], sl[2 * j], sl[2 * j + 1]);
            unpack(scw[j], sw[2 * j], sw[2 * j + 1]);
        }
#pragma unroll
        for (int j = 0; j < kCh; ++j) {
            for (int g = 0; g + 1 < k.per; ++g) s[j] += sums[(g * tr + t) * kCh + j];
            const int ch = channel<VEC>(t, tr, j);
            if (ch >= D) continue;
            if (what == 0) {
                a.part[part + ch] = s[j];
            } else {
                const float w = a.w2 ? ld_any(a.w2, a.w_dtype, ch) : 1.f, sc = a.scale_v ? ld_any(a.scale_v, a.w_dtype, ch) : a.scale;
                const float m = full ? s[j] : s[j] * ac[j];
                a.part[part + D + ch] = m * sc;
                a.part[part + 2LL * D + ch] = m * w;
                if (!full) a.part[part + 3LL * D + ch] = s[j] * sw[j] * sl[j];
            }
        }
    }
}

// Sums of the blocks' partial rows: what = 0 dw1, 1 dw2, 2 dscale over all blocks; 3 dgate over the blocks of an entry.
// ceil(D / 32) * (3 + entries) blocks, 32 x 8 threads: a thread adds every eighth partial row, four in flight, then the eight are added.
struct SumParams {
    const float *part;
    int D, blocks, entries, w_dtype, g_dtype;
    void *dpre, *dpost, *dscale, *dgate;
};
__global__ void __launch_bounds__(256) block_norm_sums(SumParams a) {
    pdl_begin();
    __shared__ float s[8][33];
    const int cols = (a.D + 31) / 32, y = blockIdx.x / cols, what = y < 3 ? y : 3, entry = y < 3 ? 0 : y - 3;
    void *out = what == 0 ? a.dpre : what == 1 ? a.dpost : what == 2 ? a.dscale : a.dgate;
    if (!out) return;
    const int c = blockIdx.x % cols * 32 + threadIdx.x, n = what < 3 ? a.blocks * a.entries : a.blocks;
    const long long stride = 4LL * a.D;
    const float *p = a.part + (long long)entry * a.blocks * stride + (long long)what * a.D + c;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < a.D) {
        int i = threadIdx.y;
        for (; i + 24 < n; i += 32) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] += p[(i + 8 * k) * stride];
        }
        for (; i < n; i += 8) v[0] += p[i * stride];
    }
    float sum = (v[0] + v[1]) + (v[2] + v[3]);
    s[threadIdx.y][threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.y || c >= a.D) return;
    for (int i = 1; i < 8; ++i) sum += s[i][threadIdx.x];
    st_any(out, what < 3 ? a.w_dtype : a.g_dtype, (long long)entry * a.D + c, sum);
}

}  // namespace bnorm
}  // namespace bissd
