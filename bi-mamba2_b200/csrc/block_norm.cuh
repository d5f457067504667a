// The norms before and after a block in one pass over a row (rms(t) = t rstd(t), rstd(t) = 1 / sqrt(mean(t^2) + eps)):
//     n = rms(x) w2,   m = scale act(gate),   r = residual + m n,   u = rms(r) w1
// and its gradients (t = u's gradient times w1, r^ = rms(r), x^ = rms(x)):
//     dr' = dr + rstd(r) (t - r^ mean(t r^)),   dresidual = dr',   dn = dr' m,   dw1 = sum_rows du r^,   dw2 = sum_rows dn x^,
//     dx = rstd(x) (dn w2 - x^ mean(dn w2 x^)),   dscale = sum_rows dr' act(gate) n,   dgate = dr' scale n act'(gate)
// Bound by the rows' bytes: each tensor is read or written once, everything between stays in registers.  A row has
// width / 8 threads with eight channels each - neighbouring ones (16-byte accesses), or where a width is no multiple of
// eight, ones a stride apart - and a block walks rows with the weights in registers, the next row's values under way while it
// sums this one's squares.  r is formed again in the backward pass, from what the forward pass read, so that no rounding of it
// enters.  Sums over rows: in registers over a block's rows, then over the blocks in a second kernel, always in one order.
#pragma once
#include <type_traits>

#include "common.cuh"

namespace bissd {
namespace bnorm {

constexpr int kCh = 8;                                           // channels a thread
constexpr int kMaxWidth = 8192;

struct Params {
    long long rows, gate_rows;                                   // gate_rows: rows of x to a row of the gate
    int D, threads_row, w_dtype, act, blocks;                    // blocks: backward, of an entry
    float scale, eps;
    long long sx, sres, sgate, sdr, sdu;                         // row strides
    const void *x, *res, *gate, *scale_v, *w2, *w1;
    void *r, *u;
    float *rstd;                                                 // [2][rows]: of x, of r
    const void *dr, *du;
    void *dx, *dres, *dgate;
    float *part;                                                 // [blocks][4][D]: dw1, dw2, dscale, dgate of a shared row
};

// Eight channels of a row as they lie in memory.
template <class T, bool VEC> struct Piece {
    using Raw = typename std::conditional<VEC, uint4[sizeof(T) / 2], T[kCh]>::type;
    Raw raw;
    __device__ __forceinline__ void load(const void *p, long long at, int t, int tr, int D) {
        const T *base = static_cast<const T *>(p) + at;
        if constexpr (VEC) {
            const bool in = t * kCh < D;
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i)
                raw[i] = in ? *(reinterpret_cast<const uint4 *>(base + t * kCh) + i) : make_uint4(0u, 0u, 0u, 0u);
        } else {
#pragma unroll
            for (int e = 0; e < kCh; ++e) raw[e] = t + e * tr < D ? base[t + e * tr] : from_f<T>(0.f);
        }
    }
    __device__ __forceinline__ void get(float (&v)[kCh]) const {
        const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
        for (int i = 0; i < kCh; ++i) v[i] = to_f<T>(e[i]);
    }
};
template <class T, bool VEC>
__device__ __forceinline__ void put(void *p, long long row, int t, int tr, int D, const float (&v)[kCh]) {
    T *base = static_cast<T *>(p) + row * D;
    if constexpr (VEC) {
        if (t * kCh >= D) return;
        union { uint4 w[sizeof(T) / 2]; T e[kCh]; } o;
#pragma unroll
        for (int i = 0; i < kCh; ++i) o.e[i] = from_f<T>(v[i]);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) *(reinterpret_cast<uint4 *>(base + t * kCh) + i) = o.w[i];
    } else {
#pragma unroll
        for (int e = 0; e < kCh; ++e)
            if (t + e * tr < D) base[t + e * tr] = from_f<T>(v[e]);
    }
}
template <bool VEC> __device__ __forceinline__ int channel(int t, int tr, int e) { return VEC ? t * kCh + e : t + e * tr; }
template <bool VEC>
__device__ __forceinline__ void weights(const void *p, int dtype, float none, int t, int tr, int D, float (&w)[kCh]) {
#pragma unroll
    for (int e = 0; e < kCh; ++e) {
        const int c = channel<VEC>(t, tr, e);
        w[e] = p ? (c < D ? ld_any(p, dtype, c) : 0.f) : none;
    }
}

// Sum over the threads of a row; every thread of the block calls.  The two buffers take turns: who writes one again has met the
// others in the call between.
template <int WARPS> __device__ __forceinline__ float row_sum(float v, float (&bufs)[2][WARPS], int &turn, int tr) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (tr == 32) return v;
    const int warp = threadIdx.x >> 5, per = tr >> 5, first = warp / per * per;
    float *buf = bufs[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) buf[warp] = v;
    __syncthreads();
    float s = 0.f;
    for (int i = 0; i < per; ++i) s += buf[first + i];
    return s;
}

// act(v) and its slope, from the hardware's 2^x and reciprocal (each within 2 ulp); 0 and 1 at the ends.
__device__ __forceinline__ void activation(int act, float v, float &a, float &slope) {
    if (act == BISSD_GATE_NONE) {
        a = v;
        slope = 1.f;
        return;
    }
    float e = v * -1.44269504f, s;
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
    if (act == BISSD_GATE_SIGMOID) {
        a = s;
        slope = s * (1.f - s);
    } else {
        a = v * s;
        slope = s * (1.f + v * (1.f - s));
    }
}

template <class T, class R, bool VEC, int THREADS>
__global__ void __launch_bounds__(THREADS, 1) block_norm_fwd(Params a) {
    pdl_begin();
    __shared__ float buf[2][THREADS / 32];
    int turn = 0;
    const int tr = a.threads_row, per = blockDim.x / tr, grp = threadIdx.x / tr, t = threadIdx.x % tr, D = a.D;
    const long long step = (long long)gridDim.x * per;
    float w2[kCh], w1[kCh], sc[kCh];
    weights<VEC>(a.w2, a.w_dtype, 1.f, t, tr, D, w2);
    weights<VEC>(a.w1, a.w_dtype, 0.f, t, tr, D, w1);
    weights<VEC>(a.scale_v, a.w_dtype, a.scale, t, tr, D, sc);
    const float inv = 1.f / D;
    Piece<T, VEC> px, pg;
    Piece<R, VEC> pr;
    auto fetch = [&](long long row) {
        if (row >= a.rows) row = a.rows - 1;
        px.load(a.x, row * a.sx, t, tr, D);
        pr.load(a.res, row * a.sres, t, tr, D);
        if (a.gate) pg.load(a.gate, (a.gate_rows > 0 ? row / a.gate_rows : row) * a.sgate, t, tr, D);
    };
    constexpr bool kAhead = VEC && THREADS <= 512;               // else the registers do not hold another row
    if (kAhead) fetch((long long)blockIdx.x * per + grp);
    for (long long base = (long long)blockIdx.x * per; base < a.rows; base += step) {
        const long long row = base + grp;
        if (!kAhead) fetch(row);
        float x[kCh], r[kCh];
        px.get(x);
        pr.get(r);
        if (a.gate) {
            float g[kCh];
            pg.get(g);
#pragma unroll
            for (int e = 0; e < kCh; ++e) {
                float act, slope;
                activation(a.act, g[e], act, slope);
                g[e] = act * sc[e] * w2[e];
            }
            if (kAhead && base + step < a.rows) fetch(row + step);
            float sx = 0.f;
#pragma unroll
            for (int e = 0; e < kCh; ++e) sx += x[e] * x[e];
            const float rx = a.w2 ? rsqrtf(row_sum(sx, buf, turn, tr) * inv + a.eps) : 1.f;
#pragma unroll
            for (int e = 0; e < kCh; ++e) r[e] += g[e] * (x[e] * rx);
            if (a.rstd && a.w2 && t == 0 && row < a.rows) a.rstd[row] = rx;
        } else {
            if (kAhead && base + step < a.rows) fetch(row + step);
            float sx = 0.f;
#pragma unroll
            for (int e = 0; e < kCh; ++e) sx += x[e] * x[e];
            const float rx = a.w2 ? rsqrtf(row_sum(sx, buf, turn, tr) * inv + a.eps) : 1.f;
#pragma unroll
            for (int e = 0; e < kCh; ++e) r[e] += sc[e] * w2[e] * (x[e] * rx);
            if (a.rstd && a.w2 && t == 0 && row < a.rows) a.rstd[row] = rx;
        }
        if (row < a.rows) put<R, VEC>(a.r, row, t, tr, D, r);
        if (a.u) {
            float sr = 0.f;
#pragma unroll
            for (int e = 0; e < kCh; ++e) sr += channel<VEC>(t, tr, e) < D ? r[e] * r[e] : 0.f;
            const float rr = rsqrtf(row_sum(sr, buf, turn, tr) * inv + a.eps);
            if (a.rstd && t == 0 && row < a.rows) a.rstd[a.rows + row] = rr;
#pragma unroll
            for (int e = 0; e < kCh; ++e) r[e] *= rr * w1[e];
            if (row < a.rows) put<T, VEC>(a.u, row, t, tr, D, r);
        }
    }
}

// entries * blocks blocks: an entry is the rows that share a gate row, where its gradient is wanted, else all of them.
template <class T, class R, bool VEC, int THREADS>
__global__ void __launch_bounds__(THREADS, 1) block_norm_bwd(Params a) {
    pdl_begin();
    __shared__ float buf[2][THREADS / 32];
    int turn = 0;
    const int tr = a.threads_row, per = blockDim.x / tr, grp = threadIdx.x / tr, t = threadIdx.x % tr, D = a.D;
    const int blk = blockIdx.x % a.blocks;
    const long long n_rows = a.rows / (gridDim.x / a.blocks), first = blockIdx.x / a.blocks * n_rows, step = (long long)a.blocks * per;
    float w2[kCh], w1[kCh], sc[kCh], d1[kCh], d2[kCh], ds[kCh], dg[kCh];
    weights<VEC>(a.w2, a.w_dtype, 1.f, t, tr, D, w2);
    weights<VEC>(a.w1, a.w_dtype, 0.f, t, tr, D, w1);
    weights<VEC>(a.scale_v, a.w_dtype, a.scale, t, tr, D, sc);
#pragma unroll
    for (int e = 0; e < kCh; ++e) d1[e] = d2[e] = ds[e] = dg[e] = 0.f;
    const float inv = 1.f / D;
    const bool row_gate = a.gate && a.gate_rows > 0;
    Piece<T, VEC> px, pg, pu;
    Piece<R, VEC> pr, pd;
    auto fetch = [&](long long i) {
        const long long row = first + (i < n_rows ? i : n_rows - 1);
        px.load(a.x, row * a.sx, t, tr, D);
        pr.load(a.res, row * a.sres, t, tr, D);
        if (a.gate) pg.load(a.gate, (row_gate ? row / a.gate_rows : row) * a.sgate, t, tr, D);
        if (a.du) pu.load(a.du, row * a.sdu, t, tr, D);
        if (a.dr) pd.load(a.dr, row * a.sdr, t, tr, D);
    };
    constexpr bool kAhead = VEC && THREADS <= 512;
    if (kAhead) fetch((long long)blk * per + grp);
    for (long long base = (long long)blk * per; base < n_rows; base += step) {
        const bool in = base + grp < n_rows;
        const long long row = first + (in ? base + grp : n_rows - 1);
        if (!kAhead) fetch(base + grp);
        float xh[kCh], r[kCh], act[kCh], m[kCh], dr[kCh], slope[kCh];
        px.get(xh);
        pr.get(r);
        const float rx = a.w2 ? a.rstd[row] : 1.f, rr = a.du ? a.rstd[a.rows + row] : 0.f;
        if (a.gate) {
            pg.get(act);
#pragma unroll
            for (int e = 0; e < kCh; ++e) activation(a.act, act[e], act[e], slope[e]);
        } else {
#pragma unroll
            for (int e = 0; e < kCh; ++e) act[e] = 1.f;
        }
#pragma unroll
        for (int e = 0; e < kCh; ++e) {
            xh[e] *= rx;
            m[e] = sc[e] * act[e];
            r[e] = (r[e] + m[e] * w2[e] * xh[e]) * rr;           // rms(r)
            dr[e] = 0.f;
        }
        if (a.dr) pd.get(dr);
        float c = 0.f, du[kCh];
        if (a.du) {
            pu.get(du);
#pragma unroll
            for (int e = 0; e < kCh; ++e) {
                if (in) d1[e] += du[e] * r[e];
                du[e] *= w1[e];
                c += du[e] * r[e];
            }
        }
        if (kAhead && base + step < n_rows) fetch(base + grp + step);
        if (a.du) {
            c = row_sum(c, buf, turn, tr) * inv;
#pragma unroll
            for (int e = 0; e < kCh; ++e) dr[e] += rr * (du[e] - r[e] * c);
        }
        if (in && a.dres) put<R, VEC>(a.dres, row, t, tr, D, dr);
        if (a.gate && a.dgate) {
            float o[kCh];
#pragma unroll
            for (int e = 0; e < kCh; ++e) {
                o[e] = dr[e] * sc[e] * w2[e] * xh[e] * slope[e];
                if (row_gate && in) dg[e] += o[e];
            }
            if (!row_gate && in) put<T, VEC>(a.dgate, row, t, tr, D, o);
        }
        float c2 = 0.f;
#pragma unroll
        for (int e = 0; e < kCh; ++e) {
            if (in) {
                ds[e] += dr[e] * act[e] * w2[e] * xh[e];
                d2[e] += dr[e] * m[e] * xh[e];
            }
            dr[e] *= m[e] * w2[e];
            c2 += dr[e] * xh[e];
        }
        if (a.w2) {
            c2 = row_sum(c2, buf, turn, tr) * inv;
#pragma unroll
            for (int e = 0; e < kCh; ++e) dr[e] = rx * (dr[e] - xh[e] * c2);
        }
        if (in && a.dx) put<T, VEC>(a.dx, row, t, tr, D, dr);
    }
    // rows side by side in this block, then one partial row a block
    extern __shared__ float dyn[];
    const long long part = (long long)blockIdx.x * 4 * D;
    float *acc[4] = {d1, d2, ds, dg};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        __syncthreads();
        if (grp > 0) {
#pragma unroll
            for (int e = 0; e < kCh; ++e) dyn[((grp - 1) * tr + t) * kCh + e] = acc[k][e];
        }
        __syncthreads();
        if (grp == 0) {
#pragma unroll
            for (int e = 0; e < kCh; ++e) {
                float s = acc[k][e];
                for (int i = 0; i + 1 < per; ++i) s += dyn[(i * tr + t) * kCh + e];
                const int ch = channel<VEC>(t, tr, e);
                if (ch < D) a.part[part + (long long)k * D + ch] = s;
            }
        }
    }
}

// Sums of the blocks' partial rows: what = 0 dw1, 1 dw2, 2 dscale over all blocks; 3 dgate over the blocks of an entry.
// ceil(D / 32) * (3 + entries) blocks, 32 x 8 threads: a thread adds every eighth partial row, then the eight are added.
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
    float v = 0.f;
    if (c < a.D)
        for (int i = threadIdx.y; i < n; i += 8) v += a.part[((long long)(entry * a.blocks + i) * 4 + what) * a.D + c];
    s[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.y || c >= a.D) return;
    for (int i = 1; i < 8; ++i) v += s[i][threadIdx.x];
    st_any(out, what < 3 ? a.w_dtype : a.g_dtype, (long long)entry * a.D + c, v);
}

}  // namespace bnorm
}  // namespace bissd
