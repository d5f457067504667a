// The causal decay attention one token after another, on CUDA cores: every type, every size, fp32 throughout.
//     S_t = e^{g_t} S_{t-1} + a_t b_t^T,    y_t = y_scale S_t^T r_t
// walked forwards with (a, b, r) = (k, v, q) gives o and, with the roles of S's two sides exchanged (v, k, dout), dq; walked
// backwards - the decay of the token after t in e^{g_t}'s place - (q, dout, k) gives dv and (dout, q, v) dk, all four from one
// kernel; dq and dk without what a token's own pair adds, e^{g_t} S_{t-1} in S_t's place (decay_finish says why).  A thread has one column of S and a part of its rows in registers; the lanes that share a column add their
// products up.  Three multiply-adds per element of S and token, two reads of shared memory (16 bytes) for every 12 of them:
// bound by those reads and the loads' instructions (670 tokens of 24 heads, 112 x 128, fp32: 102 us with outputs, 57 for states alone; the
// multiply-adds' rate would allow 20).
// A long sequence is walked in segments at once: each segment's own sum of states first (no y), the states that enter the segments
// from those (decay_chain), then the walk proper from there.
#pragma once
#include "uni_plan.cuh"

namespace bissd {
namespace uni {

constexpr int kWalkThreads = 128;

struct Vector {                                                  // one of a, b, r: (batch, token, head, inner)
    View v;
    int of_q;                                                    // its heads are those of q and k
};
struct WalkParams {
    Plan plan;
    int H, hk, I, J, lanes, reverse;                             // lanes that share a column
    Vector a, b, r;
    View g;
    int g_dtype;
    float a_scale, y_scale;
    void *y;                                                     // (tokens, H, J) contiguous, or NULL: states only
    int others;                                                  // of y: without a token's own pair
    int y_dtype;
    long long y_batch;                                           // elements of a batch row of y
    const float *init;                                           // what enters: (segments, H, ..), or NULL: zeros
    float *fin;                                                  // what leaves: (segments, H, ..), or NULL; kOthers: (sequences, H, ..), without the last token's own
    float *decay;                                                // (segments, H): the segment's whole decay, or NULL
    int si, sj;                                                  // strides of S's two sides in init and fin
    int first_decay;                                             // backwards, a whole sequence a segment: fin is one decay further back
    const int *again;                                            // flags of what is to be done, or NULL: everything
    int *status;                                                 // cleared, or NULL
};

// Tokens staged at a time, in two buffers that take turns: one tile's loads are under way while the other is walked.
__host__ __device__ inline int walk_tile(int lanes) { return lanes > 4 ? 8 : 16; }
inline size_t walk_smem(int lanes, int ipt) {
    const int tile = walk_tile(lanes), cols = kWalkThreads / lanes;
    return sizeof(float) * (2 * ((size_t)tile * 2 * lanes * (ipt + 4) + (size_t)tile * cols + 2 * tile) + (size_t)tile * cols);
}

// Y: outputs are wanted (asked at run time, the question parted the loads of every four elements: 143 us for 114, 670 tokens of 24
// heads, 112 x 128), with a token's own pair or without it.
enum { kStates = 0, kOutputs = 1, kOthers = 2 };
template <class T, int IPT, int Y> __device__ __forceinline__ void walk(const WalkParams &a, int block) {
    extern __shared__ __align__(16) float dyn[];
    const int LI = a.lanes, cols = kWalkThreads / LI, tile = walk_tile(LI), rowlen = LI * (IPT + 4);
    const int stage_len = tile * (2 * rowlen + cols + 2);
    float *ys = dyn + 2 * stage_len;
    const int jb = (a.J + cols - 1) / cols;
    const int cb = block % jb, h = block / jb % a.H, si = block / (jb * a.H);
    const Segment s = segment_or_sequence(a.plan, si);
    if (s.len == 0 || (a.again && !again(a.again, a.H, s.seq, h))) return;
    const int tid = threadIdx.x, li = tid % LI, jc = tid / LI, j = cb * cols + jc, hq = h * a.hk / a.H;
    const long long S = (long long)a.I * a.J;
    float st_[IPT];
#pragma unroll
    for (int e = 0; e < IPT; ++e) {
        const int i = li * IPT + e;
        st_[e] = a.init && i < a.I && j < a.J ? a.init[(si * (long long)a.H + h) * S + (long long)i * a.si + (long long)j * a.sj] : 0.f;
    }
    auto row = [&](const Vector &x, int t) {
        return (long long)s.batch * x.v.sb + (long long)t * x.v.sl + (long long)(x.of_q ? hq : h) * x.v.sh;
    };
    const int across = LI * IPT, la = 31 - __clz(across), lc = 31 - __clz(cols);   // powers of two
    float total = 0.f, g = 0.f;
    auto tokens = [&](int done) { return min(tile, s.len - done); };
    auto lowest = [&](int done) { return a.reverse ? s.t0 + s.len - done - tokens(done) : s.t0 + done; };
    // One value on its way to shared memory, or zero: asynchronously where it needs no conversion.
    auto put = [&](float *to, const void *from, long long at, bool in) {
        if constexpr (sizeof(T) == 4)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))),
                         "l"(static_cast<const float *>(from) + (in ? at : 0)), "r"(in ? 4 : 0) : "memory");
        else
            *to = in ? ld<T>(from, at) : 0.f;
    };
    auto fetch = [&](int done, int stage) {                      // a tile's a, r and b; its decays to a register
        if (done < s.len) {
            const int n = tokens(done), n4 = (n + 3) & ~3, first = lowest(done);   // four tokens at a time: those behind the last change nothing
            float *as = dyn + stage * stage_len, *rs = as + tile * rowlen, *bs = rs + tile * rowlen;
#pragma unroll 4
            for (int x = tid; x < n4 * across; x += kWalkThreads) {
                const int t = x >> la, i = x & (across - 1), at = t * rowlen + i / IPT * (IPT + 4) + i % IPT;
                const bool in = t < n && i < a.I;
                put(as + at, a.a.v.ptr, row(a.a, first + t) + i, in);
                if (Y != kStates) put(rs + at, a.r.v.ptr, row(a.r, first + t) + i, in);
            }
#pragma unroll 4
            for (int x = tid; x < n4 * cols; x += kWalkThreads) {
                const int t = x >> lc, c = cb * cols + (x & (cols - 1));
                const bool own = Y != kOthers || !a.fin || !s.last || first + t < s.t0 + s.len - 1;   // nothing reads what the last token adds
                put(bs + x, a.b.v.ptr, row(a.b, first + t) + c, t < n && c < a.J && own);
            }
            g = 0.f;
            const int t = first + tid + a.reverse;
            if (tid < n && !(a.reverse && s.last && t == s.t0 + s.len))
                g = ld_any(a.g.ptr, a.g_dtype, (long long)s.batch * a.g.sb + (long long)t * a.g.sl + (long long)h * a.g.sh);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto decays = [&](int stage) {                               // of the tile fetched last
        float *ds = dyn + stage * stage_len + tile * (2 * rowlen + cols);
        if (tid < tile) {
            ds[tid] = g;
            ds[tile + tid] = expf(g);
        }
    };
    fetch(0, 0);
    decays(0);
    int stage = 0;
    for (int done = 0; done < s.len; done += tile, stage ^= 1) {
        const int n = tokens(done), n4 = (n + 3) & ~3, first = lowest(done);   // lowest token of the tile
        const float *as = dyn + stage * stage_len, *rs = as + tile * rowlen, *bs = rs + tile * rowlen, *ds = bs + tile * cols, *es = ds + tile;
        fetch(done + tile, stage ^ 1);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncthreads();
        if (a.decay && tid == 0)
            for (int t = 0; t < n; ++t) total += ds[t];
        for (int u = 0; u < n4; u += 4) {
            float acc[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int t = a.reverse ? n4 - 1 - u - w : u + w;
                const float d = es[t], b = bs[t * cols + jc] * a.a_scale;
                const float4 *a4 = reinterpret_cast<const float4 *>(as + t * rowlen + li * (IPT + 4));
                const float4 *r4 = reinterpret_cast<const float4 *>(rs + t * rowlen + li * (IPT + 4));
                float sum = 0.f, sum2 = 0.f;
#pragma unroll
                for (int e = 0; e < IPT; e += 4) {
                    const float4 x = a4[e / 4];
                    auto output = [&] {
                        const float4 r = r4[e / 4];
                        sum += r.x * st_[e];
                        sum2 += r.y * st_[e + 1];
                        sum += r.z * st_[e + 2];
                        sum2 += r.w * st_[e + 3];
                    };
                    if constexpr (Y == kOthers) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) st_[e + k] *= d;
                        output();
                        st_[e] += x.x * b;
                        st_[e + 1] += x.y * b;
                        st_[e + 2] += x.z * b;
                        st_[e + 3] += x.w * b;
                    } else {
                        st_[e] = st_[e] * d + x.x * b;
                        st_[e + 1] = st_[e + 1] * d + x.y * b;
                        st_[e + 2] = st_[e + 2] * d + x.z * b;
                        st_[e + 3] = st_[e + 3] * d + x.w * b;
                        if constexpr (Y == kOutputs) output();
                    }
                }
                acc[w] = sum + sum2;
            }
            if constexpr (Y != kStates) {
                for (int o = 1; o < LI; o <<= 1) {
#pragma unroll
                    for (int w = 0; w < 4; ++w) acc[w] += __shfl_xor_sync(0xffffffffu, acc[w], o);
                }
                if (li == 0) {
#pragma unroll
                    for (int w = 0; w < 4; ++w) ys[(a.reverse ? n4 - 1 - u - w : u + w) * cols + jc] = acc[w] * a.y_scale;
                }
            }
        }
        if (done + tile < s.len) decays(stage ^ 1);
        __syncthreads();                                         // the tile has been read, and ys is written: the next barrier lets it be again
        if constexpr (Y != kStates) {
            for (int x = tid; x < n * cols; x += kWalkThreads) {
                const int t = x >> lc, c = cb * cols + (x & (cols - 1));
                if (c < a.J)
                    st_any(a.y, a.y_dtype, (long long)s.batch * a.y_batch + ((long long)(first + t) * a.H + h) * a.J + c, ys[x]);
            }
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (a.fin && (Y != kOthers || s.last)) {
        const long long to = Y == kOthers ? s.seq : si;
        if (a.first_decay) {
            const float d = expf(ld_any(a.g.ptr, a.g_dtype, (long long)s.batch * a.g.sb + (long long)s.t0 * a.g.sl + (long long)h * a.g.sh));
#pragma unroll
            for (int e = 0; e < IPT; ++e) st_[e] *= d;
        }
#pragma unroll
        for (int e = 0; e < IPT; ++e) {
            const int i = li * IPT + e;
            if (i < a.I && j < a.J) a.fin[(to * (long long)a.H + h) * S + (long long)i * a.si + (long long)j * a.sj] = st_[e];
        }
    }
    if (a.decay && cb == 0 && tid == 0) a.decay[si * (long long)a.H + h] = expf(total);
}

template <class T, int IPT, int Y> __global__ void __launch_bounds__(kWalkThreads, 4) decay_walk(WalkParams a) {
    pdl_begin();
    if (a.status && blockIdx.x == 0 && threadIdx.x == 0) *a.status = 0;
    walk<T, IPT, Y>(a, blockIdx.x);
}
// What is done again: the walk of a forward pass, or the three of a backward pass at once.  Mostly there is nothing to do, and then a launch costs
// its latency and the blocks it starts: no more than are resident, which take the walks' blocks in turn.  Eight rows a thread.
constexpr int kAgainRows = 8;
template <class T> __global__ void __launch_bounds__(kWalkThreads, 4)
decay_walks_again(const __grid_constant__ WalkParams out, const __grid_constant__ WalkParams dk, const __grid_constant__ WalkParams dq, int out_blocks, int dk_blocks,
                  int blocks) {
    pdl_begin();
    if (!out.again[0]) return;
    for (int x = blockIdx.x; x < blocks; x += gridDim.x) {
        const int block = x - out_blocks;
        if (block < 0) walk<T, kAgainRows, kOutputs>(out, x);
        else if (block < dk_blocks) walk<T, kAgainRows, kOthers>(dk, block);
        else walk<T, kAgainRows, kOthers>(dq, block - dk_blocks);
        __syncthreads();                                         // shared memory has been read
    }
}

// The states that enter the segments, from each segment's own sum (in its place): forwards run = D run + own, written before it is
// added to; backwards the same from the last segment on.  Also the state after the last segment (forwards), or the gradient of
// the initial state: that of the state after the first token, times the first token's decay (backwards).
// A thread has an element of one (sequence, head).   `per` elements a state.
struct ChainParams {
    Plan plan;
    int H, per, reverse, nseq;
    const float *start;                                          // (sequences, H, per), or NULL
    float *states;                                               // (segments, H, per): own sums in, entering states out
    const float *decay;                                          // (segments, H)
    float *end;                                                  // (sequences, H, per), or NULL
    int first_decay;                                             // backwards: `end` is one decay further back
    View g;
    int g_dtype;
};
template <int VEC> struct Quad { float v[VEC]; };
template <int VEC> __device__ __forceinline__ Quad<VEC> quad_ld(const float *p) {
    Quad<VEC> q;
    if constexpr (VEC == 4) {
        const float4 f = *reinterpret_cast<const float4 *>(p);
        q.v[0] = f.x; q.v[1] = f.y; q.v[2] = f.z; q.v[3] = f.w;
    } else {
        q.v[0] = *p;
    }
    return q;
}
template <int VEC> __device__ __forceinline__ void quad_st(float *p, const Quad<VEC> &q) {
    if constexpr (VEC == 4) *reinterpret_cast<float4 *>(p) = make_float4(q.v[0], q.v[1], q.v[2], q.v[3]);
    else *p = q.v[0];
}
template <int VEC> __global__ void __launch_bounds__(256) decay_chain(ChainParams a) {
    pdl_begin();
    const int blocks = (a.per + 256 * VEC - 1) / (256 * VEC);
    const int e = (blockIdx.x % blocks * 256 + threadIdx.x) * VEC, h = blockIdx.x / blocks % a.H, seq = blockIdx.x / (blocks * a.H);
    if (e >= a.per) return;
    const long long of_seq = ((long long)seq * a.H + h) * a.per + e;
    const int2 f = segments(a.plan, seq);
    Quad<VEC> run = {};
    if (a.start) run = quad_ld<VEC>(a.start + of_seq);
    for (int u0 = 0; u0 < f.y; u0 += 4) {                        // four segments' values under way at a time
        Quad<VEC> own[4];
        float d[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int u = min(u0 + k, f.y - 1), i = f.x + (a.reverse ? f.y - 1 - u : u);
            own[k] = quad_ld<VEC>(a.states + ((long long)i * a.H + h) * a.per + e);
            d[k] = a.decay[(long long)i * a.H + h];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int u = u0 + k, i = f.x + (a.reverse ? f.y - 1 - u : u);
            if (u < f.y) {
                quad_st<VEC>(a.states + ((long long)i * a.H + h) * a.per + e, run);
#pragma unroll
                for (int x = 0; x < VEC; ++x) run.v[x] = run.v[x] * d[k] + own[k].v[x];
            }
        }
    }
    if (a.end) {
        if (a.first_decay && f.y > 0) {
            const Segment s = segment(a.plan, f.x);
            const float d = expf(ld_any(a.g.ptr, a.g_dtype, (long long)s.batch * a.g.sb + (long long)s.t0 * a.g.sl + (long long)h * a.g.sh));
#pragma unroll
            for (int x = 0; x < VEC; ++x) run.v[x] *= d;
        }
        quad_st<VEC>(a.end + of_seq, run);
    }
}

// What the per-head gradients leave: dq and dk summed over the heads that share them, with the tokens' own pairs, which the walks leave
// out: scale sum_h (do_t.v_t) times k_t or q_t (a warp for a token and head of q); and what a token's decay gets from its own place,
// into = q.dq and from = k.dk (a pair of tokens s < t counts +1 at t and -1 at s; a warp for a token and head).  A token's own pair would be
// in both of these, and the larger it is beside the others the fewer digits their difference would have.  The second reads again what the first has read: together, one warp's heads waited for one another
// (89 us, 15 so: 670 tokens, 24 heads of 2, kdim 112).
struct FinishParams {
    int L, H, hk, N, P, nseq;
    long long tokens;
    float scale;
    View q, k, v, dout;
    const int *bounds;                                           // packed: the sequences' tokens are bounds[0] ... bounds[nseq] - 1; or NULL
    const float *dqh, *dkh;                                      // (tokens, H, N), others' part
    void *dq, *dk;                                               // (tokens, hk, N)
    float *into, *from;                                          // (tokens, H)
    const int *again;                                            // as in WalkParams
};
template <class T> __global__ void __launch_bounds__(256) decay_finish(FinishParams a) {
    pdl_begin();
    if (a.again && !a.again[0]) return;
    const int lane = threadIdx.x & 31, R = a.H / a.hk;
    const long long sums = a.tokens * a.hk, all = sums + (a.into ? a.tokens * a.H : 0);
    for (long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < all; i += (long long)gridDim.x * 8) {
        const long long w = i < sums ? i : i - sums, tok = i < sums ? w / a.hk : w / a.H, b = tok / a.L, t = tok % a.L;
        const int m = i < sums ? (int)(w % a.hk) : (int)(w % a.H) / R;
        const bool in = !a.bounds || (t >= a.bounds[0] && t < a.bounds[a.nseq]);
        if (a.again) {
            if (!in) continue;
            int seq = (int)b;
            if (a.bounds) {                                      // the last sequence that begins at t or before it and is not behind it
                int lo = 0, hi = a.nseq;
                while (hi - lo > 1) {
                    const int mid = (lo + hi) / 2;
                    if (a.bounds[mid] <= t) lo = mid;
                    else hi = mid;
                }
                seq = lo;
            }
            if (!again(a.again, a.H, seq, m * R)) continue;
        }
        const long long at = b * a.q.sb + t * a.q.sl + m * a.q.sh, kt = b * a.k.sb + t * a.k.sl + m * a.k.sh;
        if (i < sums) {
            const long long from = w * R * a.N;
            float own = 0.f;
            if (in) {
                for (int r = 0; r < R; ++r) {
                    const long long vt = b * a.v.sb + t * a.v.sl + (long long)(m * R + r) * a.v.sh,
                                    dt = b * a.dout.sb + t * a.dout.sl + (long long)(m * R + r) * a.dout.sh;
#pragma unroll 4
                    for (int p = lane; p < a.P; p += 32) own += ld<T>(a.v.ptr, vt + p) * ld<T>(a.dout.ptr, dt + p);
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) own += __shfl_xor_sync(0xffffffffu, own, o);
                own *= a.scale;
            }
            for (int n = lane; n < a.N; n += 32) {
                float sq = 0.f, sk = 0.f;
                if (in) {
#pragma unroll 4
                    for (int r = 0; r < R; ++r) {
                        sq += a.dqh[from + (long long)r * a.N + n];
                        sk += a.dkh[from + (long long)r * a.N + n];
                    }
                    sq = fmaf(own, ld<T>(a.k.ptr, kt + n), sq);
                    sk = fmaf(own, ld<T>(a.q.ptr, at + n), sk);
                }
                st<T>(a.dq, w * a.N + n, sq);
                st<T>(a.dk, w * a.N + n, sk);
            }
            continue;
        }
        if (!in) continue;                                       // of no use to anyone
        float x = 0.f, y = 0.f;
#pragma unroll 4
        for (int n = lane; n < a.N; n += 32) {
            x += ld<T>(a.q.ptr, at + n) * a.dqh[w * a.N + n];
            y += ld<T>(a.k.ptr, kt + n) * a.dkh[w * a.N + n];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            x += __shfl_xor_sync(0xffffffffu, x, o);
            y += __shfl_xor_sync(0xffffffffu, y, o);
        }
        if (lane == 0) {
            a.into[w] = x;
            a.from[w] = y;
        }
    }
}

// dg_t: everything that flows from tokens before t (or the initial state) to t and those after (or the final state) = what crosses
// the segment's right end + into - from of the tokens t ... there.  What crosses is a product of two states, so rounding does not pile
// up over more than one segment.  At a sequence's end these are the final state without what its last token adds, which crosses no decay, and
// the final state's gradient; all that flows from the last token is that part, and is not counted either.  A block for a (segment, head).
// Off by 3e-7 to 9e-7 of its norm, whether decays are e^-0.005 or e^-12 a token (with own pairs on both sides 6e-7 to 8e-4, and 1e-2 where these are
// large: 90 and 130 tokens).
struct DecayGradParams {
    Plan plan;
    int H, per, g_dtype, out_dtype, L;
    const float *into, *from, *enter, *denter;                   // states entering each segment from the left, gradients from the right
    const float *final_, *dfinal;                                // (sequences, H, per), final_ without the last tokens' own; dfinal NULL: zeros
    View g;
    void *dg;                                                    // (tokens, H)
    const int *again;                                            // as in WalkParams
};
__global__ void __launch_bounds__(256) decay_dg(DecayGradParams a) {
    pdl_begin();
    __shared__ double part[8], carry;
    const int h = blockIdx.x % a.H, si = blockIdx.x / a.H, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (a.again && !a.again[0]) return;
    const Segment s = segment_or_sequence(a.plan, si);
    if (s.len == 0 || (a.again && !again(a.again, a.H, s.seq, h))) return;
    const int end = s.t0 + s.len;
    double cross = 0.0;
    if (!s.last || a.dfinal) {
        const long long here = ((long long)si * a.H + h) * a.per;
        const float *x = s.last ? a.final_ + ((long long)s.seq * a.H + h) * a.per : a.enter + here + (long long)a.H * a.per;
        const float *y = s.last ? a.dfinal + ((long long)s.seq * a.H + h) * a.per : a.denter + here;
        for (int e = tid; e < a.per; e += 256) cross += (double)x[e] * y[e];
        if (!s.last) cross *= expf(ld_any(a.g.ptr, a.g_dtype, (long long)s.batch * a.g.sb + (long long)end * a.g.sl + (long long)h * a.g.sh));
    }
    for (int o = 16; o > 0; o >>= 1) cross += __shfl_xor_sync(0xffffffffu, cross, o);
    if (lane == 0) part[warp] = cross;
    __syncthreads();
    if (tid == 0) {
        double c = 0.0;
        for (int w = 0; w < 8; ++w) c += part[w];
        carry = c;
    }
    __syncthreads();
    for (int hi = end; hi > s.t0; hi -= 256) {                   // from the right, thread 0 the last token
        const int t = hi - 1 - tid;
        const long long at = ((long long)s.batch * a.L + t) * a.H + h;
        double v = t >= s.t0 ? (double)a.into[at] - (s.last && t == end - 1 ? 0.f : a.from[at]) : 0.0;
        for (int o = 1; o < 32; o <<= 1) {
            const double u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        if (lane == 31) part[warp] = v;
        __syncthreads();
        double before = carry;
        for (int w = 0; w < warp; ++w) before += part[w];
        if (t >= s.t0) st_any(a.dg, a.out_dtype, at, (float)(before + v));
        __syncthreads();
        if (tid == 255) carry = before + v;
        __syncthreads();
    }
}

// One decay for each head: the sum of its tokens' gradients, in a fixed order.  bounds: of packed sequences, or NULL.
__global__ void __launch_bounds__(1024) decay_dg_heads(const float *dg, long long tokens, int H, void *out, int dtype, const int *bounds, int nseq) {
    pdl_begin();
    __shared__ double part[32];
    double v = 0.0;
    const int first = bounds ? bounds[0] : 0;
    const long long end = bounds ? bounds[nseq] : tokens;
    for (long long t = threadIdx.x; t < end; t += 1024)
        if (t >= first) v += dg[t * H + blockIdx.x];
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 1; w < 32; ++w) v += part[w];
    st_any(out, dtype, blockIdx.x, (float)v);
}

}  // namespace uni
}  // namespace bissd
