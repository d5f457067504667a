// The causal decay attention on the tensor cores (bf16 or fp16: T), in chunks of 128 tokens.  With c_t the sum of the chunk's log decays up to
// and with token t, and S the state that enters the chunk,
//     o_t = scale [ e^{c_t} S^T q_t + sum_{s <= t} e^{c_t - c_s} (q_t.k_s) v_s ],    S' = e^{c_end} S + sum_s k_s (e^{c_end - c_s} v_s)^T
// so a chunk is four products of 128 rows; only S' waits for the chunk before it.
//   decay_states   walks the chunks of one head with S in registers and writes what enters each: the k v^T products alone
//   decay_chunks   all chunks at once, given the states
// Heads of v are taken 64 columns at a time: with the same weights, v's parts are heads of their own that share q, k and g.  Head sizes
// that fill no tile are completed by the loads with zeros.  Log decays count in powers of two and no lower than 2^-200 a token, which
// fp32 has no number for: -inf never meets +inf.  Factors that reach to a chunk's ends are 2 to the power of a sum that starts there, and
// and those between two tokens of sums over what lies between them, so that a strong decay elsewhere in the chunk costs no digits.
// Products take operands of T: states, pairs and weighted rows are rounded to it.  In fp16 they may be out of its range where inputs and
// outputs are not.  An operand that is no number leaves no number in every sum that it enters, so the kernels look at their fp32 sums alone,
// and heads of sequences where one is none are done again by uni_walk.cuh's kernels, which leave at once where there are none
// (one more launch forward, three backward; with the looking 265 -> 286 us for both passes of 8 x 2048 tokens of 24 heads).
#pragma once
#include "tc_tma.cuh"
#include "uni_plan.cuh"
#include "vec.cuh"

namespace bissd {
namespace unitc {

using namespace tc;
using uni::Plan;
using uni::Segment;

constexpr int kQ = 128;                                          // tokens a chunk
constexpr int kP = 64;                                           // columns of v a tile
constexpr int kSlab = kQ * 128;                                  // 128 rows of 64 values
constexpr int kErrDecay = 0x2000;                                // status word: a wait of these kernels ran out

struct Heads {
    int H, hk, N, P, PB;                                         // PB: tiles of v's columns
    View g;
    int g_dtype;
    float log_scale;                                             // log2 of scale > 0
};

// Log2 decays of four tokens in a row, lane l's tokens 4 l ... 4 l + 3 of the chunk; zeros behind the chunk's end.  They are kept
// as loaded until they are summed: what asks for them does not wait for them.
struct Decays {
    float v[4];
    uint32_t raw[4];
    __device__ __forceinline__ void load(const Heads &a, int batch, int t0, int len, int h, int lane) {
        const long long at = (long long)batch * a.g.sb + (long long)t0 * a.g.sl + (long long)h * a.g.sh;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = lane * 4 + i;
            raw[i] = 0;
            if (t < len) {
                if (a.g_dtype == BISSD_F32) raw[i] = __ldg(static_cast<const uint32_t *>(a.g.ptr) + at + t * a.g.sl);
                else raw[i] = __ldg(static_cast<const unsigned short *>(a.g.ptr) + at + t * a.g.sl);
            }
        }
    }
    __device__ __forceinline__ void log2(const Heads &a) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float g = a.g_dtype == BISSD_F16 ? __half2float(__ushort_as_half((unsigned short)raw[i]))
                                                   : __uint_as_float(a.g_dtype == BISSD_F32 ? raw[i] : raw[i] << 16);
            const float x = g * 1.44269504f;
            v[i] = x < -200.f ? -200.f : x;                      // what is no number stays none
        }
    }
    // Sums up to and with each token, from the first of its W lanes on.  What is needed between two tokens is made of sums over what lies
    // between them, not of one such sum less another: where tokens empty the state one over a chunk comes to 25600, and a step of fp32 is 2^-9 there.
    // (Sums of 32 tokens are subtracted where they are at most 64.)
    template <int W = 32> __device__ __forceinline__ void prefix(float (&c)[4], int lane) const {
        c[0] = v[0];
#pragma unroll
        for (int i = 1; i < 4; ++i) c[i] = c[i - 1] + v[i];
        float sum = c[3];
#pragma unroll
        for (int o = 1; o < W; o <<= 1) {
            const float u = __shfl_up_sync(0xffffffffu, sum, o);
            if ((lane & (W - 1)) >= o) sum += u;
        }
        const float before = __shfl_up_sync(0xffffffffu, sum, 1);
        if (lane & (W - 1)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] += before;
        }
    }
    // Sums of the tokens behind each, up to the last of its W lanes.
    template <int W = 32> __device__ __forceinline__ void suffix(float (&c)[4], int lane) const {
        c[3] = 0.f;
#pragma unroll
        for (int i = 2; i >= 0; --i) c[i] = c[i + 1] + v[i + 1];
        float sum = c[0] + v[0];
#pragma unroll
        for (int o = 1; o < W; o <<= 1) {
            const float u = __shfl_down_sync(0xffffffffu, sum, o);
            if ((lane & (W - 1)) + o < W) sum += u;
        }
        const float behind = __shfl_down_sync(0xffffffffu, sum, 1);
        if ((lane & (W - 1)) < W - 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] += behind;
        }
    }
};

// Rows of a tile behind the sequence's end: a packed neighbour's, of whatever values, become zeros.
__device__ __forceinline__ void clear_rows(uint8_t *slab, int from, int tid, int threads) {
    for (int i = from * 8 + tid; i < kQ * 8; i += threads) *reinterpret_cast<uint4 *>(slab + i * 16) = zero8();
}

// A weight f as f1 + f2 of type T, and eight values of T times it in one rounding: v f1 + (v f2) as a multiply-add.
template <class T> struct PairOf;
template <> struct PairOf<__nv_bfloat16> { using type = __nv_bfloat162; };
template <> struct PairOf<__half> { using type = __half2; };
template <class T> __device__ __forceinline__ uint32_t halves(float f) {
    const float hi = to_f<T>(from_f<T>(f));
    return pack2<T>(hi, f - hi);
}
template <class T> __device__ __forceinline__ uint4 weighted(const uint4 &row, uint32_t f) {
    using T2 = typename PairOf<T>::type;
    const uint32_t f1 = __byte_perm(f, f, 0x1010), f2 = __byte_perm(f, f, 0x3232);
    uint32_t e[4] = {row.x, row.y, row.z, row.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const T2 v = *reinterpret_cast<const T2 *>(&e[q]);
        const T2 o = __hfma2(v, *reinterpret_cast<const T2 *>(&f1), __hmul2(v, *reinterpret_cast<const T2 *>(&f2)));
        e[q] = *reinterpret_cast<const uint32_t *>(&o);
    }
    return make_uint4(e[0], e[1], e[2], e[3]);
}
__device__ __forceinline__ float both(vec::f2 v) {
    float a, b;
    vec::unpack(v, a, b);
    return a + b;
}

// ---- the states that enter the chunks ------------------------------------------------------------------------------------
// Forwards S' as above; backwards (v the outputs' gradient, k the queries) the gradient that enters each chunk from its right,
// G' = e^{c_end} G + sum_t q_t (scale e^{c_t} do_t)^T.  A block walks the chunks of one (segment, head, 64 columns), S or G in
// registers (a row n and 32 columns a thread).  k's and v's rows come by TMA a chunk ahead.  Eight warps weight v's in place and keep S;
// the ninth issues loads and MMAs, the tenth makes the weights and stores the tiles, and they meet at mbarriers alone: a step is S's
// way to shared memory, one product's latency, its way back and the weighting.  (The weighting in the product's shadow, from rows
// loaded to registers, made it longer: the loads from tensor memory then waited for those rows.)
// Two blocks an SM, to the byte: the barriers lie behind the tiles, and there is no other shared memory.
// EXACT: the weighted row is given to the tensor cores in three 16-bit parts, each what is left of those before, so that the states
// that leave the library are fp32's.  The tiles that the other kernels read are 16-bit in any case: they meet 16-bit factors.  The parts
// lie side by side and take one product of 192 columns, which reads k once, and meet again as three sums: shared memory bounds this
// (as three products of 64 columns, in two rounds, 190 us for 142: 512 chunks of 32 heads, 128 x 64 states, sums alone; the walk
// proper, not EXACT, takes 124 for 0.54 GB).  The third part goes
// where v's rows came, in front of the others or behind them in turn, and k has one buffer: its next rows come while v's are weighted.
struct StatesParams {
    Heads h;
    Plan seg, chunk;
    int reverse, by_seq, tiles;                                  // by_seq: init and fin hold a state a sequence, not a segment
    const float *init;
    float *fin, *decay;                                          // decay: (segments, H) the segment's whole decay, or NULL
    int *status;
    int clear;                                                   // the status, by the first block: any wait of another takes far longer to run out
    int *again;                                                  // fp16: flags of what is to be done again, cleared; or NULL
    int *bad;                                                    // fp16, EXACT: by blocks, whether what leaves is out of fp16's range; or NULL
};
// The thread's tile stores so far have read their shared memory.
__device__ __forceinline__ void tma_store_read() {
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}
struct StatesShared {
    uint64_t full[2], full_v[2], ready, done, weights, stored, unused;
    uint32_t tmem;
    int fail, loads, loads_v, bad;                               // fail: the first wait that ran out; loads asked for
    float decay[2];                                              // of a chunk, 2^c_end
    alignas(16) uint32_t w[kQ];                                  // of a chunk's rows: f1 and f2, or EXACT fp32
};
constexpr int kStatesThreads = 320;
inline size_t states_smem(int NT, bool exact) { return (exact ? NT / 64 + 5 : 2 * (NT / 64) + 3) * (size_t)kSlab + sizeof(StatesShared); }

template <class T, int NT, bool EXACT> __global__ void __launch_bounds__(kStatesThreads, 2)
decay_states(StatesParams a, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmTiles) {
    pdl_begin();
    if (a.clear && blockIdx.x == 0 && threadIdx.x == 0) *a.status = 0;
    constexpr bool kNarrow = std::is_same<T, __half>::value;     // what lies between inputs and outputs may be out of T's range
    if (kNarrow && a.again && blockIdx.x == 0 && threadIdx.x == 0) a.again[0] = 0;
    constexpr int kSlabs = NT / 64;
    extern __shared__ __align__(1024) uint8_t dyn[];
    // two stages of k, two of weighted rows, S.  EXACT: one of k, v's rows, two parts, v's rows, S
    uint8_t *smK = dyn, *smV = smK + (EXACT ? 1 : 2) * kSlabs * kSlab, *smS = smV + (EXACT ? 4 : 2) * kSlab;
    StatesShared &sh = *reinterpret_cast<StatesShared *>(smS + kSlab);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int pb = blockIdx.x % a.h.PB, h = blockIdx.x / a.h.PB % a.h.H, si = blockIdx.x / (a.h.PB * a.h.H), hq = h * a.h.hk / a.h.H;
    const Segment s = uni::segment(a.seg, si);
    if (kNarrow && a.bad && tid == 0 && s.len == 0) a.bad[blockIdx.x] = 0;
    if (s.len == 0) return;                                      // packed: fewer segments than there could be
    if (kNarrow && a.again && tid == 0 && pb == 0 && s.idx == 0) a.again[1 + (long long)s.seq * a.h.H + h] = 0;
    if (smem_u32(dyn) & 1023) {                                  // the swizzled tiles' alignment, which nothing else here sees to
        if (tid == 0) atomicExch(a.status, kErrDecay + 4);
        return;
    }
    const int nc = ceil_div(s.len, kQ);
    auto place = [&](int i) { return a.reverse ? nc - 1 - i : i; };        // chunk of the segment at step i
    auto length = [&](int i) { return min(kQ, s.len - place(i) * kQ); };
    volatile int *fail = &sh.fail;
    if (warp == 0) tmem_alloc(&sh.tmem, EXACT ? 256 : 64);
    if (tid == 256) {
        mbar_init(&sh.full[0], 1);
        mbar_init(&sh.full[1], 1);
        mbar_init(&sh.full_v[0], 1);
        mbar_init(&sh.full_v[1], 1);
        mbar_init(&sh.ready, 8);
        mbar_init(&sh.done, 1);
        mbar_init(&sh.weights, 1);
        mbar_init(&sh.stored, 1);
        sh.fail = sh.bad = 0;
        fence_mbar_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    bool ok = true;
    if (warp == 8) {
        auto load = [&](int i) {
            const int st = EXACT ? 0 : i & 1, t = s.t0 + place(i) * kQ;
            mbar_expect_tx(&sh.full[st], (kSlabs + !EXACT) * kSlab);
            for (int j = 0; j < kSlabs; ++j) tma_load4(smK + (st * kSlabs + j) * kSlab, &tmK, j * 64, hq, t, s.batch, &sh.full[st]);
            if (!EXACT) tma_load4(smV + st * kSlab, &tmV, pb * kP, h, t, s.batch, &sh.full[st]);
            if (EXACT && i + 1 < nc)                             // the next one's as far as L2: their load waits for the buffer
                for (int j = 0; j < kSlabs; ++j)
                    asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];" ::"l"(&tmK), "r"(j * 64), "r"(hq),
                                 "r"(s.t0 + place(i + 1) * kQ), "r"(s.batch) : "memory");
        };
        auto load_v = [&](int i) {                               // EXACT
            const int st = i & 1;
            mbar_expect_tx(&sh.full_v[st], kSlab);
            tma_load4(smV + st * 3 * kSlab, &tmV, pb * kP, h, s.t0 + place(i) * kQ, s.batch, &sh.full_v[st]);
        };
        int loads = 1, loads_v = EXACT ? min(nc, 2) : 0;
        if (lane == 0) {
            load(0);
            for (int i = 0; i < loads_v; ++i) load_v(i);
        }
        constexpr uint32_t idesc = instr_desc(AbFmt<T>::v, true, true, EXACT ? 3 * kP : kP);
        for (int i = 0; i < nc && ok; ++i) {
            const int st = EXACT ? 0 : i & 1;
            if (!EXACT && i + 1 < nc) {                          // the stage was read by the MMAs of the step before
                if (i > 0) ok = ws_wait_warp(&sh.done, (i - 1) & 1, fail, 1);
                if (ok && lane == 0) load(i + 1);
                loads += ok;
            }
            ok = ok && ws_wait_warp(&sh.full[st], (EXACT ? i : i >> 1) & 1, fail, 2) && ws_wait_warp(&sh.ready, i & 1, fail, 3);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
                const uint8_t *v = smV + (i & 1) * kSlab;
#pragma unroll 1
                for (int kk = 0; kk < kQ / 16; ++kk)             // where NT is 64, rows 64 ... 127 are the first 64 again: products of no use
                    umma(tmem, smem_desc(smem_u32(smK + st * kSlabs * kSlab) + kk * 2048, NT == 64 ? 0 : kSlab, 1024),
                         smem_desc(smem_u32(v) + kk * 2048, kSlab, 1024), idesc, kk > 0);
                umma_commit(&sh.done);
            }
            __syncwarp();
            if (EXACT && i + 1 < nc) {
                ok = ws_wait_warp(&sh.done, i & 1, fail, 1);
                if (!ok) break;
                if (lane == 0) load(i + 1);
                ++loads;
                if (i + 2 < nc) {
                    if (lane == 0) load_v(i + 2);
                    ++loads_v;
                }
            }
        }
        if (lane == 0) {
            sh.loads = loads;
            sh.loads_v = loads_v;
        }
    } else if (warp == 9) {
        const int c0 = uni::segments(a.chunk, s.seq).x + s.idx * (a.seg.seg / kQ);
        Decays d;
        uint32_t f[4];
        float whole = 0.f, total = 0.f;
        auto ask = [&](int i) {
            if (i < nc) d.load(a.h, s.batch, s.t0 + place(i) * kQ, length(i), h, lane);
        };
        auto make = [&]() {                                      // the weights of what was asked for last
            float c[4];
            d.log2(a.h);
            if (a.reverse) {
                d.prefix(c, lane);
                whole = __shfl_sync(0xffffffffu, c[3], 31);
            } else {
                d.suffix(c, lane);
                whole = __shfl_sync(0xffffffffu, c[0] + d.v[0], 0);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float v = exp2f(a.reverse ? c[k] + a.h.log_scale : c[k]);
                f[k] = EXACT ? __float_as_uint(v) : halves<T>(v);
            }
        };
        auto give = [&](int i) {                                 // to the others, as chunk i's
            *reinterpret_cast<uint4 *>(&sh.w[lane * 4]) = make_uint4(f[0], f[1], f[2], f[3]);
            if (lane == 0) sh.decay[i & 1] = exp2f(whole);
            total += whole;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.weights);
        };
        ask(0);
        make();
        give(0);
        ask(1);
        if (nc > 1) make();
        ask(2);
        for (int i = 0; i < nc; ++i) {
            ok = ws_wait_warp(&sh.ready, i & 1, fail, 9);       // the next one cannot come before this warp's weights: none is missed
            if (!ok) break;
            if (i + 1 < nc) give(i + 1);
            if (a.tiles && elect_one()) {
                tma_store2(&tmTiles, smS, 0, (((c0 + place(i)) * a.h.H + h) * a.h.PB + pb) * NT);
                tma_store_read();                                // S's tile may be written again
                mbar_arrive(&sh.stored);
            }
            __syncwarp();
            if (i + 2 < nc) {
                make();
                ask(i + 3);
            }
        }
        if (a.decay && ok && pb == 0 && lane == 0) a.decay[(long long)si * a.h.H + h] = exp2f(total);
        if (a.tiles && elect_one()) tma_store_wait();
        __syncwarp();
    } else {
        const uint32_t swz = (tid >> 3) * 128 + (((tid & 7) ^ ((tid >> 3) & 7)) << 4);   // the thread's piece of a tile, + 4096 k
        auto weigh = [&](uint8_t *v, int len) {                  // rows times f1 + f2, in their place
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint4 row = weighted<T>(*reinterpret_cast<const uint4 *>(v + swz + k * 4096), sh.w[(tid >> 3) + k * 32]);
                // rows behind the sequence's end may be of another, and no numbers
                *reinterpret_cast<uint4 *>(v + swz + k * 4096) = (tid >> 3) + k * 32 < len ? row : zero8();
            }
        };
        constexpr float kUp = std::is_same<T, __half>::value ? 2048.f : 1.f;   // fp16: keeps the second and third part out of its small numbers
        auto parts = [&](int i, int len) {                       // chunk i's weighted rows: the third part in their place
            uint8_t *third = smV + (i & 1) * 3 * kSlab + swz, *first = smV + kSlab + swz;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float f = __uint_as_float(sh.w[(tid >> 3) + k * 32]);
                const uint4 row = (tid >> 3) + k * 32 < len ? *reinterpret_cast<const uint4 *>(third + k * 4096) : zero8();
                uint32_t e[4] = {row.x, row.y, row.z, row.w}, o1[4], o2[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float x, y, hx, hy;
                    unpack2<T>(e[q], x, y);
                    x *= f;
                    y *= f;
                    o1[q] = pack2<T>(x, y);
                    unpack2<T>(o1[q], hx, hy);
                    x = (x - hx) * kUp;
                    y = (y - hy) * kUp;
                    o2[q] = pack2<T>(x, y);
                    unpack2<T>(o2[q], hx, hy);
                    e[q] = pack2<T>((x - hx) * kUp, (y - hy) * kUp);
                }
                *reinterpret_cast<uint4 *>(first + k * 4096) = make_uint4(o1[0], o1[1], o1[2], o1[3]);
                *reinterpret_cast<uint4 *>(first + kSlab + k * 4096) = make_uint4(o2[0], o2[1], o2[2], o2[3]);
                *reinterpret_cast<uint4 *>(third + k * 4096) = make_uint4(e[0], e[1], e[2], e[3]);
            }
        };
        const int n = (warp & 3) * 32 + lane, half = warp >> 2, col = pb * kP + half * 32;
        const long long at = (((long long)(a.by_seq ? s.seq : si) * a.h.H + h) * a.h.N + n) * a.h.P + col;
        float S[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) S[j] = a.init && n < a.h.N && col + j < a.h.P ? a.init[at + j] : 0.f;
        const uint32_t tl = tmem_lane_base(tmem) + half * 32;
        auto arrive = [&] {                                      // what this warp wrote is there, what it read of tensor memory is read
            fence_async_smem();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.ready);
        };
        auto prepare = [&](int i) {                              // chunk i's rows
            const int st = i & 1;
            if (!ws_wait_warp(&sh.weights, i & 1, fail, 4) || !ws_wait_warp(&sh.full[st], (i >> 1) & 1, fail, 6)) return false;
            weigh(smV + st * kSlab, length(i));
            if (a.seg.packed && length(i) < kQ)
                for (int j = 0; j < kSlabs; ++j) clear_rows(smK + (st * kSlabs + j) * kSlab, length(i), tid, 256);
            return true;
        };
        if constexpr (!EXACT) ok = prepare(0);
        for (int i = 0; i < nc && ok; ++i) {
            const int st = i & 1;
            float now;
            if constexpr (EXACT) {
                ok = ws_wait_warp(&sh.weights, i & 1, fail, 4) && ws_wait_warp(&sh.full_v[st], (i >> 1) & 1, fail, 10);
                if (!ok) break;
                parts(i, length(i));
            }
            now = sh.decay[st];
            if (a.tiles) {                                       // what enters this chunk
                if (i > 0) ok = ws_wait_warp(&sh.stored, (i - 1) & 1, fail, 5);
                if (!ok) break;
                if (n < NT) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float e[8] = {S[8 * j], S[8 * j + 1], S[8 * j + 2], S[8 * j + 3], S[8 * j + 4], S[8 * j + 5], S[8 * j + 6], S[8 * j + 7]};
                        *reinterpret_cast<uint4 *>(smS + n * 128 + (((half * 4 + j) ^ (n & 7)) << 4)) = pack8<T>(e);
                    }
                }
            }
            if (EXACT && a.seg.packed && length(i) < kQ) {
                ok = ws_wait_warp(&sh.full[0], i & 1, fail, 6);
                if (!ok) break;
                for (int j = 0; j < kSlabs; ++j) clear_rows(smK + j * kSlab, length(i), tid, 256);
            }
            arrive();
            ok = ws_wait_warp(&sh.done, i & 1, fail, 8);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int j0 = 0; j0 < 32; j0 += 16) {
                float x[16];
                tmem_ld16(tl + j0, x);
                if constexpr (EXACT) {                           // the buffer that comes first or last has the third part
                    float y[16], z[16];
                    tmem_ld16(tl + kP + j0, y);
                    tmem_ld16(tl + 2 * kP + j0, z);
                    const float fx = st ? 1.f : 1.f / (kUp * kUp), fy = st ? 1.f / kUp : 1.f, fz = st ? 1.f / (kUp * kUp) : 1.f / kUp;
#pragma unroll
                    for (int j = 0; j < 16; ++j) S[j0 + j] = fmaf(S[j0 + j], now, kUp == 1.f ? x[j] + (y[j] + z[j]) : fmaf(x[j], fx, fmaf(y[j], fy, z[j] * fz)));
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) S[j0 + j] = fmaf(S[j0 + j], now, x[j]);
                }
            }
            if constexpr (!EXACT)
                if (i + 1 < nc) ok = prepare(i + 1);
        }
        if (ok && a.fin && n < a.h.N) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (col + j < a.h.P) a.fin[at + j] = S[j];
            if (kNarrow && a.bad) {                              // a row times a weight above 1, in a part of 16 bits
                float none = 0.f;
#pragma unroll
                for (int j = 0; j < 32; ++j) none = fmaf(S[j], 0.f, none);
                if (none != 0.f) sh.bad = 1;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (sh.fail) {                                               // a wait of any role ran out: leave nothing in flight
        if (tid == 0) atomicExch(a.status, kErrDecay + 0x10 + sh.fail);
        if (warp == 8 && elect_one()) {
            drain_mmas(&sh.unused);
            drain_loads(sh.full, EXACT ? 1 : 2, sh.loads);
            drain_loads(sh.full_v, 2, sh.loads_v);
        }
        __syncthreads();
    }
    if (kNarrow && a.bad && tid == 0) a.bad[blockIdx.x] = sh.bad;
    if (warp == 0) tmem_dealloc(tmem, EXACT ? 256 : 64);
}

// ---- the outputs -----------------------------------------------------------------------------------------------------
// A block has one chunk of one head of q and k, and walks `vpc` of the tiles of v that share them: Q, K and their product stay, in
// shared and tensor memory, and per tile come v's rows and the state.  The product, weighted by the decays and rounded to T (it
// meets v's T), takes K's place in shared memory.  Where a block of 32 x 32 lies below the diagonal, the weight is a row factor times a
// column factor, both counted from the block's last column and at most 1; on the diagonal it is one 2^x an element, of the difference of two
// sums over 32 tokens at most, or where these are above 64 of a sum that starts at the row's token and takes in a token a column (a chain:
// 234 us for 211 if always so).  A warp has
// 32 rows and half of the columns up to the diagonal, in units of 16.
// Two blocks an SM: one's loads and element-wise work run under the other's MMAs.  Bound by memory where rows are long: 512 chunks of
// 32 heads, 128 x 64 states, 1.05 GB in 216 us (4.7 TB/s).  Stores from registers, without the way through shared memory, took 244
// us, 512 threads a block 264.
struct ChunksParams {
    Heads h;
    Plan chunk;
    int vpc, parts;                                              // tiles of v a block, blocks a (chunk, head of q)
    void *o;                                                     // (tokens, H, P) contiguous
    int *status;
    uni::Again again;                                            // fp16
};
inline size_t chunks_smem(int NT) { return 1024 + (size_t)(NT / 64) * kSlab + 2 * (size_t)kSlab + (size_t)kSlab + (size_t)NT * 128; }

template <class T, int NT> __global__ void __launch_bounds__(256, 2)
decay_chunks(ChunksParams a, const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
             const __grid_constant__ CUtensorMap tmS) {
    pdl_begin();
    constexpr bool kNarrow = std::is_same<T, __half>::value;     // what lies between inputs and outputs may be out of T's range
    if constexpr (kNarrow) uni::do_again_states(a.again, 1, 256);
    constexpr int kSlabs = NT / 64, kTables = 8;                 // heads whose tables are made at a time, one a warp
    extern __shared__ __align__(1024) uint8_t dyn[];
    __shared__ uint64_t bar_qk, bar_v, bar_s, done, done_s, unused;
    __shared__ uint32_t tmem_slot;
    __shared__ __align__(16) float gs[kTables][kQ], upto[kTables][kQ], below[kTables][kQ];   // log2 decays; their sums in t's 32 up to t; 2^(sum in s' 32 behind s)
    __shared__ float between[kTables][4][4];                     // [1 + b][q]: sums of the 32s behind the b-th and before the q-th
    uint8_t *smQ = smem_align1024(dyn), *smK = smQ + kSlabs * kSlab, *smV = smK + 2 * kSlab, *smS = smV + kSlab;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int part = blockIdx.x % a.parts, m = blockIdx.x / a.parts % a.h.hk, ci = blockIdx.x / (a.parts * a.h.hk);
    const Segment s = uni::segment(a.chunk, ci);
    if (s.len == 0) return;
    const int R = a.h.H / a.h.hk, v0 = part * a.vpc, nv = min(a.vpc, R * a.h.PB - v0), h0 = m * R + v0 / a.h.PB;
    int h = h0, pb = v0 - v0 / a.h.PB * a.h.PB;                  // of the present tile
    const int heads = (pb + nv + a.h.PB - 1) / a.h.PB;
    auto load_v = [&](int h, int pb) {
        mbar_expect_tx(&bar_v, kSlab);
        tma_load4(smV, &tmV, pb * kP, h, s.t0, s.batch, &bar_v);
    };
    auto load_s = [&](int h, int pb) {
        mbar_expect_tx(&bar_s, NT * 128);
        tma_load2(smS, &tmS, 0, ((ci * a.h.H + h) * a.h.PB + pb) * NT, &bar_s);
    };
    Decays next;                                                 // this warp's head of the next kTables
    auto ask = [&](int k) {
        if (k < heads) next.load(a.h, s.batch, s.t0, s.len, h0 + k, lane);
    };
    auto table = [&](int k) {
        if (k >= heads) return;
        float c[4], w[4];
        next.log2(a.h);
        next.prefix<8>(c, lane);
        next.suffix<8>(w, lane);
        float sum = 0.f;
#pragma unroll
        for (int b = 0; b < 3; ++b) {
            const float of = __shfl_sync(0xffffffffu, c[3], 8 * b + 7);
            sum += b >= lane >> 2 && b < (lane & 3) ? of : 0.f;
        }
        if (lane < 16) between[warp][lane >> 2][lane & 3] = sum;
        *reinterpret_cast<float4 *>(&gs[warp][lane * 4]) = make_float4(next.v[0], next.v[1], next.v[2], next.v[3]);
        *reinterpret_cast<float4 *>(&upto[warp][lane * 4]) = make_float4(c[0], c[1], c[2], c[3]);
        *reinterpret_cast<float4 *>(&below[warp][lane * 4]) = make_float4(exp2f(w[0]), exp2f(w[1]), exp2f(w[2]), exp2f(w[3]));
    };
    ask(warp);
    if (warp == 0) tmem_alloc(&tmem_slot, 256);
    if (tid == 32) {
        mbar_init(&bar_qk, 1);
        mbar_init(&bar_v, 1);
        mbar_init(&bar_s, 1);
        mbar_init(&done, 1);
        mbar_init(&done_s, 1);
        fence_mbar_init();
        mbar_expect_tx(&bar_qk, 2 * kSlabs * kSlab);
        for (int j = 0; j < kSlabs; ++j) {
            tma_load4(smQ + j * kSlab, &tmQ, j * 64, m, s.t0, s.batch, &bar_qk);
            tma_load4(smK + j * kSlab, &tmK, j * 64, m, s.t0, s.batch, &bar_qk);
        }
        load_s(h, pb);
        load_v(h, pb);
    }
    table(warp);
    ask(kTables + warp);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot, tl = tmem_lane_base(tmem);  // columns: 0 q.k, 128 inside the chunk, 192 from the state
    int loads_v = 1, loads_s = 1;
    bool ok = true;
    if (warp == 0 && elect_one()) {
        ok = mbar_wait(&bar_qk, 0);
        if (ok) {
            constexpr uint32_t idesc = instr_desc(AbFmt<T>::v, false, false, kQ);
#pragma unroll 1
            for (int kk = 0; kk < NT / 16; ++kk)
                umma(tmem, smem_desc(smem_u32(smQ + kk / 4 * kSlab) + kk % 4 * 32, 16, 1024),
                     smem_desc(smem_u32(smK + kk / 4 * kSlab) + kk % 4 * 32, 16, 1024), idesc, kk > 0 ? 1u : 0u);
            umma_commit(&done);
        }
    }
    if (ok) ok = mbar_wait(&done, 0);
    ok = __syncthreads_and(ok);                                  // k's rows are dead: the weighted pairs take their place
    tc_fence_after();
    const int r32 = warp & 3, t = r32 * 32 + lane, half = warp >> 2;   // this thread: row t, 32 columns of each output tile
    const int u0 = half * (r32 + 1), u1 = u0 + r32 + 1;          // and units u0 ... u1 - 1 of 16 weighted pairs
    auto pair_at = [&](int u) { return smK + (u >> 2) * kSlab + t * 128; };
    auto piece = [&](int u, int j) { return (((u & 3) * 2 + j) ^ (t & 7)) << 4; };
    if (ok && half == 1)
        for (int u = 2 * (r32 + 1); u < 8; ++u)                  // above the diagonal
            for (int j = 0; j < 2; ++j) *reinterpret_cast<uint4 *>(pair_at(u) + piece(u, j)) = zero8();
    T *out = static_cast<T *>(a.o) + ((long long)s.batch * a.chunk.L + s.t0 + (tid >> 3)) * a.h.H * a.h.P;   // the first of the rows this thread writes
    const long long row32 = 32LL * a.h.H * a.h.P;
    for (int i = 0; i < nv && ok; ++i) {
        const int k = h - h0, h1 = h + (pb + 1 == a.h.PB), pb1 = pb + 1 == a.h.PB ? 0 : pb + 1;   // and the next tile's
        if (i > 0 && k % kTables == 0 && pb == 0) {
            __syncthreads();                                     // the last tables have been read
            table(k + warp);
            ask(k + kTables + warp);
            __syncthreads();
        }
        if (warp == 0 && elect_one()) {                          // from the state: Q S
            ok = mbar_wait(&bar_s, i & 1);
            if (ok) {
                tc_fence_after();
                constexpr uint32_t idesc = instr_desc(AbFmt<T>::v, false, true, kP);
#pragma unroll 1
                for (int kk = 0; kk < NT / 16; ++kk)
                    umma(tmem + 192, smem_desc(smem_u32(smQ + kk / 4 * kSlab) + kk % 4 * 32, 16, 1024),
                         smem_desc(smem_u32(smS) + kk * 2048, NT * 128, 1024), idesc, kk > 0 ? 1u : 0u);
                umma_commit(&done_s);
            }
        }
        const float *g = gs[k % kTables], *c = upto[k % kTables];
        const float ct = c[t] + a.h.log_scale;
        const bool strong = fabsf(c[r32 * 32 + 31]) > 64.f;      // differences of sums lack digits
        {
            uint32_t raw[16];
            tmem_ld16_nowait(tl + u0 * 16, raw);
            for (int u = u0; u < u1; ++u) {
                vec::f2 x[8];
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = vec::pack(__uint_as_float(raw[2 * j]), __uint_as_float(raw[2 * j + 1]));
                if (u + 1 < u1) tmem_ld16_nowait(tl + (u + 1) * 16, raw);
                const int cb = u >> 1;
                if (cb < r32) {
                    const float rt = exp2f(ct + between[k % kTables][1 + cb][r32]);
                    const vec::f2 rt2 = vec::pack(rt, rt);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float4 f = *reinterpret_cast<const float4 *>(below[k % kTables] + u * 16 + j * 4);
                        x[2 * j] = vec::mul2(x[2 * j], vec::mul2(vec::pack(f.x, f.y), rt2));
                        x[2 * j + 1] = vec::mul2(x[2 * j + 1], vec::mul2(vec::pack(f.z, f.w), rt2));
                    }
                } else {
                    const int td = t - u * 16;                   // columns up to it; what is behind it may be no number
                    if (!strong) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float2 f = *reinterpret_cast<const float2 *>(c + u * 16 + j * 2);
                            float lo, hi;
                            vec::unpack(x[j], lo, hi);
                            lo *= ex2_approx(ct - f.x);
                            hi *= ex2_approx(ct - f.y);
                            x[j] = vec::pack(2 * j <= td ? lo : 0.f, 2 * j + 1 <= td ? hi : 0.f);
                        }
                    } else {
                        float e = td > 15 ? a.h.log_scale : -INFINITY;   // from the unit's end
                        for (int x = u * 16 + 16; x <= t; ++x) e += g[x];
#pragma unroll
                        for (int j = 7; j >= 0; --j) {
                            const float2 f = *reinterpret_cast<const float2 *>(g + u * 16 + j * 2);
                            float lo, hi;
                            vec::unpack(x[j], lo, hi);
                            if (2 * j + 1 == td) e = a.h.log_scale;
                            hi *= ex2_approx(e);
                            e += f.y;
                            if (2 * j == td) e = a.h.log_scale;
                            lo *= ex2_approx(e);
                            e += f.x;
                            x[j] = vec::pack(2 * j <= td ? lo : 0.f, 2 * j + 1 <= td ? hi : 0.f);
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    uint4 o;
                    o.x = vec::narrow<T>(x[4 * j]); o.y = vec::narrow<T>(x[4 * j + 1]);
                    o.z = vec::narrow<T>(x[4 * j + 2]); o.w = vec::narrow<T>(x[4 * j + 3]);
                    *reinterpret_cast<uint4 *>(pair_at(u) + piece(u, j)) = o;
                }
            }
            if (r32 == 0 && half == 1)                           // the output's tile lay there
                for (int u = 2; u < 4; ++u)
                    for (int j = 0; j < 2; ++j) *reinterpret_cast<uint4 *>(pair_at(u) + piece(u, j)) = zero8();
        }
        if (a.chunk.packed && s.len < kQ) {
            ok = ok && mbar_wait(&bar_v, i & 1);
            if (ok) clear_rows(smV, s.len, tid, 256);
        }
        fence_async_smem();
        ok = __syncthreads_and(ok);
        if (!ok) break;
        if (warp == 0 && elect_one()) {                          // inside the chunk: the weighted pairs times v
            ok = mbar_wait(&bar_v, i & 1);
            if (ok) {
                tc_fence_after();
                constexpr uint32_t idesc = instr_desc(AbFmt<T>::v, false, true, kP);
#pragma unroll 1
                for (int kk = 0; kk < kQ / 16; ++kk)
                    umma(tmem + 128, smem_desc(smem_u32(smK + kk / 4 * kSlab) + kk % 4 * 32, 16, 1024),
                         smem_desc(smem_u32(smV) + kk * 2048, kSlab, 1024), idesc, kk > 0 ? 1u : 0u);
                umma_commit(&done);
            }
        }
        if (i + 1 < nv) {                                        // the state's tile is long read; v's rows when all is done
            if (tid == 32) ok = mbar_wait(&done_s, i & 1);
            if (tid == 32 && ok) load_s(h1, pb1);
            ++loads_s;
        }
        if (ok) ok = mbar_wait(&done, (i + 1) & 1) && mbar_wait(&done_s, i & 1);
        if (i + 1 < nv) {
            if (tid == 32 && ok) load_v(h1, pb1);
            ++loads_v;
        }
        tc_fence_after();
        // o = inside + scale e^{c_t} from the state; whole rows leave through the first slab of the weighted pairs
        if (ok) {
            const float f = exp2f(ct + between[k % kTables][0][r32]);
            float x[32], y[32], none = 0.f;
            tmem_ld32(tl + 128 + half * 32, x);
            tmem_ld32(tl + 192 + half * 32, y);
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
                float e[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    e[q] = fmaf(y[j + q], f, x[j + q]);
                    if constexpr (kNarrow) none = fmaf(e[q], 0.f, none);
                }
                *reinterpret_cast<uint4 *>(smK + t * 128 + (((half * 4 + (j >> 3)) ^ (t & 7)) << 4)) = pack8<T>(e);
            }
            if (kNarrow && none != 0.f && t < s.len) uni::do_again(a.again, s.seq, h, 1);
        }
        tc_fence_before();
        ok = __syncthreads_and(ok);
        if (!ok) break;
        const int col = pb * kP + (tid & 7) * 8;
        if (col < a.h.P) {
            T *o = out + h * a.h.P + col;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int r = (tid >> 3) + q * 32;
                if (r < s.len) *reinterpret_cast<uint4 *>(o + q * row32) = *reinterpret_cast<const uint4 *>(smK + r * 128 + (((tid & 7) ^ (r & 7)) << 4));
            }
        }
        __syncthreads();                                         // the slab is the pairs' again
        tc_fence_after();
        h = h1;
        pb = pb1;
    }
    ok = __syncthreads_and(ok);
    if (!ok && tid == 0) atomicExch(a.status, kErrDecay + 2);
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        if (!ok && elect_one()) {                                // leave nothing in flight
            drain_mmas(&unused);
            drain_loads(&bar_qk, 1, 1);
            drain_loads(&bar_v, 1, loads_v);
            drain_loads(&bar_s, 1, loads_s);
        }
        __syncwarp();
        tmem_dealloc(tmem, 256);
    }
}

// ---- the gradients ------------------------------------------------------------------------------------------------------
// All chunks at once, given what enters each from the left (S) and from the right (G, the gradient of the state behind the chunk).
// With w_ts = scale e^{c_t - c_s} for s <= t, p = w (q.k) and d = w (do.v):
//     dv_s = sum_t p_ts do_t + e^{c_end - c_s} G^T k_s        dk_s = sum_t d_ts q_t + G (e^{c_end - c_s} v_s)
//     dq_t = sum_s d_ts k_s + S (scale e^{c_t} do_t)
//     dg_t = e^{c_end} S.G  +  sum_{t' >= t} scale e^{c_t'} do_t'.S^T q_t'  +  sum_{s < t} e^{c_end - c_s} v_s.G^T k_s  +  sum_{s < t <= t'} d_t's q_t'.k_s
// - every pair of places before and from t on: past and future of the chunk, past and its tokens, its tokens and the future, tokens
// among themselves; the last as sums over rows less sums over columns of the same fp32 products, without tokens' own pairs, which would be
// in both and, where decays are strong, nearly all of them.  Everything is laid out with s along the rows (lanes): p and d then are operands of dv and dk as they lie, and d of dq
// read the other way.  p goes back to tensor memory, d to shared memory.  A block has a chunk and a head of q and k, and walks (its
// part of) the heads of v that share them, dq and dk adding up in tensor memory; v and do come a tile ahead, the states while the pairs
// are weighted, and the products of d run under the next tile's first ones, when nobody waits for them.  Ten of the sixteen warps have weights to make, six lie above the
// diagonal: one of these makes the next head's tables, one sums dg, one issues the products, and together they weight v.  A tile's
// products (3300 cycles, most from shared memory) and its arithmetic (7000) take turns: 128 chunks of 24 heads, 128 x 64 states, 162 us on 128
// SMs.  The loops of products are not unrolled: a shorter body ran 180 -> 170 us.
struct GradsParams {
    Heads h;
    Plan chunk;
    int vpc, parts;                                              // tiles of v a block (whole heads), blocks a (chunk, head of q)
    void *dq, *dk, *dv;                                          // contiguous
    float *part;                                                 // parts > 1: (2, parts, tokens, hk, N), dq and dk
    long long tokens;
    void *dg;                                                    // DG: (tokens, H)
    int dg_dtype;
    int *status;
    uni::Again again;                                            // fp16
};
inline size_t grads_smem(int NT) { return 1024 + 2 * (size_t)(NT / 64) * kSlab + 4 * (size_t)kSlab + 3 * (size_t)kSlab + 2 * (size_t)NT * 128; }

// A from tensor memory: 128 lanes, two 16-bit values of K a column.
__device__ __forceinline__ void umma_tmem(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        :
        : "r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        :
        : "r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
          "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}

template <class T, int NT, bool DG> __global__ void __launch_bounds__(512, 1)
decay_grads(GradsParams a, const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
            const __grid_constant__ CUtensorMap tmD, const __grid_constant__ CUtensorMap tmS, const __grid_constant__ CUtensorMap tmG) {
    pdl_begin();
    constexpr bool kNarrow = std::is_same<T, __half>::value;     // what lies between inputs and outputs may be out of T's range
    if constexpr (kNarrow) uni::do_again_states(a.again, a.h.H / a.h.hk, 512);
    constexpr int kSlabs = NT / 64, kT = 512;
    constexpr int kTables = 2, kHelp = 3, kIssue = 7, kSums = 11;   // warps above the diagonal
    extern __shared__ __align__(1024) uint8_t dyn[];
    struct Table {                                               // of a head; two take turns
        float g[kQ], ws[kQ];                                     // log2 of a token's decay; e^{c_end - c_s}
        uint32_t wv[kQ], wd[kQ];                                 // that and scale e^{c_t} in halves, for v and do
        float above[kQ], beside[3][kQ];                          // weights of blocks of 32 x 32: 2^(c at the end of s' 32 - c_s), scale 2^(c_t - c at the end of the q-th 32)
        float whole[4];                                          // c_end
    };
    __shared__ uint64_t bar_qk, bar_v[2], bar_s, done_1, done_a, done_b, unused;
    __shared__ uint32_t tmem_slot;
    __shared__ __align__(16) Table tables[2];
    __shared__ __align__(16) float rowsum[4][kQ], colsum[4][kQ], past[4][kQ], future[4][kQ], cross[16];
    uint8_t *smQ = smem_align1024(dyn), *smK = smQ + kSlabs * kSlab, *smV = smK + kSlabs * kSlab, *smD = smV + 2 * kSlab, *smE = smD + 2 * kSlab,
            *smN = smE + kSlab, *smS = smN + 2 * kSlab, *smG = smS + NT * 128;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int part = blockIdx.x % a.parts, m = blockIdx.x / a.parts % a.h.hk, ci = blockIdx.x / (a.parts * a.h.hk);
    const Segment sg = uni::segment(a.chunk, ci);
    if (sg.len == 0) return;
    const int len = sg.len, R = a.h.H / a.h.hk, v0 = part * a.vpc, nv = min(a.vpc, R * a.h.PB - v0);
    const bool tail = a.chunk.packed && len < kQ;                // rows of another sequence lie behind this one's
    const int h0 = m * R + v0 / a.h.PB;                          // the block's first head; it starts with the head's first tile
    auto load_v = [&](int i, int h, int pb) {
        const int b = i & 1;
        mbar_expect_tx(&bar_v[b], 2 * kSlab);
        tma_load4(smV + b * kSlab, &tmV, pb * kP, h, sg.t0, sg.batch, &bar_v[b]);
        tma_load4(smD + b * kSlab, &tmD, pb * kP, h, sg.t0, sg.batch, &bar_v[b]);
    };
    auto load_s = [&](int h, int pb) {
        const int row = ((ci * a.h.H + h) * a.h.PB + pb) * NT;
        mbar_expect_tx(&bar_s, 2 * NT * 128);
        tma_load2(smS, &tmS, 0, row, &bar_s);
        tma_load2(smG, &tmG, 0, row, &bar_s);
    };
    auto table = [&](Table &to, Decays &next) {                  // one warp
        float c[4], q[4];
        next.log2(a.h);
        next.prefix<8>(c, lane);
        next.suffix<8>(q, lane);
        const int own = lane >> 3;                               // 32 tokens of four
        float sums[4];                                           // theirs
#pragma unroll
        for (int b = 0; b < 4; ++b) sums[b] = __shfl_sync(0xffffffffu, c[3], 8 * b + 7);
        auto four = [&](float *o, auto f) { *reinterpret_cast<float4 *>(o + lane * 4) = make_float4(f(0), f(1), f(2), f(3)); };
        four(to.g, [&](int k) { return next.v[k]; });
        four(to.above, [&](int k) { return ex2_approx(q[k]); });
        float rest = 0.f, head = a.h.log_scale;                  // behind the lane's 32 tokens, and before them
#pragma unroll
        for (int b = 1; b < 4; ++b) rest += b > own ? sums[b] : 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = ex2_approx(q[k] + rest);
        four(to.ws, [&](int k) { return q[k]; });
        *reinterpret_cast<uint4 *>(to.wv + lane * 4) = make_uint4(halves<T>(q[0]), halves<T>(q[1]), halves<T>(q[2]), halves<T>(q[3]));
#pragma unroll
        for (int b = 2; b >= 0; --b) {                           // of use in the blocks behind the b-th
            four(to.beside[b], [&](int k) { return ex2_approx(c[k] + head); });
            head += b < own ? sums[b] : 0.f;
        }
        auto wd = [&](int k) { return halves<T>(ex2_approx(c[k] + head)); };
        *reinterpret_cast<uint4 *>(to.wd + lane * 4) = make_uint4(wd(0), wd(1), wd(2), wd(3));
        if (lane == 0) to.whole[0] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    };
    if (warp == 0) tmem_alloc(&tmem_slot, 512);
    if (tid == 32) {
        mbar_init(&bar_qk, 1);
        mbar_init(&bar_v[0], 1);
        mbar_init(&bar_v[1], 1);
        mbar_init(&bar_s, 1);
        mbar_init(&done_1, 1);
        mbar_init(&done_a, 1);
        mbar_init(&done_b, 1);
        fence_mbar_init();
        mbar_expect_tx(&bar_qk, 2 * kSlabs * kSlab);
        for (int j = 0; j < kSlabs; ++j) {
            tma_load4(smQ + j * kSlab, &tmQ, j * 64, m, sg.t0, sg.batch, &bar_qk);
            tma_load4(smK + j * kSlab, &tmK, j * 64, m, sg.t0, sg.batch, &bar_qk);
        }
        load_v(0, h0, 0);
        load_s(h0, 0);
        if (nv > 1) load_v(1, h0 + (a.h.PB == 1), a.h.PB == 1 ? 0 : 1);
    }
    if (warp == kTables) {
        Decays d;
        d.load(a.h, sg.batch, sg.t0, len, h0, lane);
        table(tables[0], d);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // tensor memory: 0 q.k, then p as T (64 columns); 64 dv inside the chunk; 128 do.v, then dv from the future; 192 S^T q; dq; dk
    const uint32_t tmem = tmem_slot, tl = tmem_lane_base(tmem);
    constexpr uint32_t cOwn = 64, cFar = 128, cOut = 192, cQ = 256, cK = 256 + NT;
    int loads_v = nv > 1 ? 2 : 1, loads_s = 1;
    bool ok = mbar_wait(&bar_qk, 0);
    const int quad = warp & 3, cg = warp >> 2, s = quad * 32 + lane;   // this thread: row s; columns t of 32 cg ...; 16 of dv's 64
    if (ok && tail)
        for (int j = 0; j < kSlabs; ++j) {
            clear_rows(smQ + j * kSlab, len, tid, kT);
            clear_rows(smK + j * kSlab, len, tid, kT);
        }
    float through = 0.f;                                         // this thread's part of S.G
    const long long token = (long long)sg.batch * a.chunk.L + sg.t0;
    // 16-byte pieces of a tile of 128 x 64, two a thread; the issuing warp's are another's
    const int reps = warp == kIssue ? 0 : warp == kHelp ? 2 : 1;
    auto pieces = [&](auto f) {
        for (int r = 0; r < reps; ++r) {
            f(tid + r * (kIssue - kHelp) * 32);
            f(tid + r * (kIssue - kHelp) * 32 + kT);
        }
    };
    auto put_dv = [&](int i, int h, int pb) {                    // tile i's from v's place
        const uint8_t *from = smV + (i & 1) * kSlab;
        T *dv = static_cast<T *>(a.dv) + (token * a.h.H + h) * a.h.P + pb * kP;
        const int row_values = a.h.H * a.h.P;
        pieces([&](int x) {
            const int r = x >> 3, col = (x & 7) * 8;
            if (r < len && pb * kP + col < a.h.P)
                *reinterpret_cast<uint4 *>(dv + (long long)r * row_values + col) =
                    *reinterpret_cast<const uint4 *>(from + r * 128 + (((x & 7) ^ (r & 7)) << 4));
        });
    };
    auto from_chunk = [&]() {                                    // dq and dk of the chunk's own pairs; one thread
        constexpr uint32_t iq = instr_desc(AbFmt<T>::v, true, true, NT), ik = instr_desc(AbFmt<T>::v, false, true, NT);
        const uint32_t q0 = smem_u32(smQ), k0 = smem_u32(smK), n0 = smem_u32(smN);
#pragma unroll 1
        for (int kk = 0; kk < kQ / 16; ++kk) {
            umma(tmem + cQ, smem_desc(n0 + kk * 2048, kSlab, 1024), smem_desc(k0 + kk * 2048, kSlab, 1024), iq, 1u);
            umma(tmem + cK, smem_desc(n0 + kk / 4 * kSlab + kk % 4 * 32, 16, 1024), smem_desc(q0 + kk * 2048, kSlab, 1024), ik, 1u);
        }
        umma_commit(&done_b);
    };
    int h = h0, pb = 0;                                          // of tile i
    for (int i = 0; i < nv; ++i) {
        const bool first = pb == 0, last = pb + 1 == a.h.PB;     // tiles of a head
        const int h1 = h + last, pb1 = last ? 0 : pb + 1;        // of the next one
        const Table &tb = tables[(h - h0) & 1];
        uint8_t *sV = smV + (i & 1) * kSlab, *sD = smD + (i & 1) * kSlab;
        if (tail) {
            ok = ok && mbar_wait(&bar_v[i & 1], (i >> 1) & 1);
            if (ok) {
                clear_rows(sV, len, tid, kT);
                clear_rows(sD, len, tid, kT);
            }
            fence_async_smem();
            ok = __syncthreads_and(ok);
            if (!ok) break;
        }
        if (warp == kIssue && elect_one()) {                     // q.k and do.v of all pairs, rows s
            ok = ok && mbar_wait(&bar_v[i & 1], (i >> 1) & 1);
            if (ok) {
                tc_fence_after();
                constexpr uint32_t idesc = instr_desc(AbFmt<T>::v, false, false, kQ);
#pragma unroll 1
                for (int kk = 0; kk < NT / 16; ++kk)
                    umma(tmem, smem_desc(smem_u32(smK + kk / 4 * kSlab) + kk % 4 * 32, 16, 1024),
                         smem_desc(smem_u32(smQ + kk / 4 * kSlab) + kk % 4 * 32, 16, 1024), idesc, kk > 0 ? 1u : 0u);
#pragma unroll 1
                for (int kk = 0; kk < 4; ++kk)
                    umma(tmem + 128, smem_desc(smem_u32(sV) + kk * 32, 16, 1024), smem_desc(smem_u32(sD) + kk * 32, 16, 1024), idesc, kk > 0 ? 1u : 0u);
                umma_commit(&done_1);
                if (i > 0) from_chunk();                         // of the tile before: here nothing waits for them
            }
        }
        if (ok && i > 0) put_dv(i - 1, h0 + (i - 1) / a.h.PB, pb == 0 ? a.h.PB - 1 : pb - 1);
        if (ok) ok = mbar_wait(&bar_v[i & 1], (i >> 1) & 1);
        if (ok) {
            pieces([&](int x) {                                  // scale e^{c_t} do_t beside do_t
                *reinterpret_cast<uint4 *>(smE + x * 16) = weighted<T>(*reinterpret_cast<const uint4 *>(sD + x * 16), tb.wd[x >> 3]);
            });
            ok = mbar_wait(&done_1, i & 1);
        }
        tc_fence_after();
        const bool some = cg >= quad;                            // a block on the diagonal or below it
        float x[32], y[32];
        if (ok && some) {
            tmem_ld32(tl + cg * 32, x);
            tmem_ld32(tl + 128 + cg * 32, y);
        }
        tc_fence_before();
        asm volatile("bar.sync %0, 128;" ::"r"(1 + quad) : "memory");   // p goes where these 32 rows' q.k was
        tc_fence_after();
        if (ok && i > 0) ok = mbar_wait(&done_b, (i - 1) & 1);   // d of the tile before has been read
        if (ok) {
            uint8_t *drow = smN + (cg >> 1) * kSlab + s * 128;   // rows of 64 t, 16-byte pieces swizzled
            uint32_t p[16];
            float of_row = 0.f, of_column = 0.f;                 // for dg: d (q.k) over this row, over column 32 cg + lane
            if (some) {
                const float fs = tb.above[s];
                const float4 *f4 = reinterpret_cast<const float4 *>(cg == quad ? tb.g + cg * 32 : tb.beside[quad] + cg * 32);
                vec::f2 sum = vec::pack(0.f, 0.f);
                float c = -INFINITY;                             // on the diagonal c_t - c_s, summed from s on
                auto weight = [&](int j, float g) {
                    c = j == lane ? a.h.log_scale : c + g;
                    return ex2_approx(c);
                };
#pragma unroll
                for (int j0 = 0; j0 < 32; j0 += 8) {
                    uint32_t d[4];
#pragma unroll
                    for (int j = j0; j < j0 + 8; j += 4) {
                        const float4 f = f4[j / 4];
                        const vec::f2 x0 = vec::pack(x[j], x[j + 1]), x1 = vec::pack(x[j + 2], x[j + 3]);
                        vec::f2 w0, w1, others0 = x0, others1 = x1;
                        if (cg == quad) {
                            const float e0 = weight(j, f.x), e1 = weight(j + 1, f.y), e2 = weight(j + 2, f.z), e3 = weight(j + 3, f.w);
                            w0 = vec::pack(e0, e1);
                            w1 = vec::pack(e2, e3);
                            if constexpr (DG) {                  // a token's own pair crosses no decay
                                others0 = vec::pack(j == lane ? 0.f : x[j], j + 1 == lane ? 0.f : x[j + 1]);
                                others1 = vec::pack(j + 2 == lane ? 0.f : x[j + 2], j + 3 == lane ? 0.f : x[j + 3]);
                            }
                        } else {
                            const vec::f2 fs2 = vec::pack(fs, fs);
                            w0 = vec::mul2(vec::pack(f.x, f.y), fs2);
                            w1 = vec::mul2(vec::pack(f.z, f.w), fs2);
                        }
                        const vec::f2 y0 = vec::mul2(vec::pack(y[j], y[j + 1]), w0), y1 = vec::mul2(vec::pack(y[j + 2], y[j + 3]), w1);
                        p[j / 2] = vec::narrow<T>(vec::mul2(x0, w0));
                        p[j / 2 + 1] = vec::narrow<T>(vec::mul2(x1, w1));
                        d[(j - j0) / 2] = vec::narrow<T>(y0);
                        d[(j - j0) / 2 + 1] = vec::narrow<T>(y1);
                        if constexpr (DG) {
                            const vec::f2 z0 = vec::mul2(others0, y0), z1 = vec::mul2(others1, y1);
                            sum = vec::add2(sum, vec::add2(z0, z1));
                            vec::unpack(z0, x[j], x[j + 1]);
                            vec::unpack(z1, x[j + 2], x[j + 3]);
                        }
                    }
                    *reinterpret_cast<uint4 *>(drow + ((((cg & 1) * 4 + j0 / 8) ^ (s & 7)) << 4)) = make_uint4(d[0], d[1], d[2], d[3]);
                }
                if constexpr (DG) {
                    of_row = both(sum);
                    auto value = [&](auto k) { return x[decltype(k)::value]; };
                    of_column = warp_sums<32>(value, lane);
                }
            } else {
                const int light = (quad == 3 ? 3 : quad - 1) + cg;   // of six warps
                for (int x = light * 32 + lane; x < kQ * 8; x += 6 * 32) {   // e^{c_end - c_s} v_s in v_s' place
                    uint4 *v = reinterpret_cast<uint4 *>(sV + x * 16);
                    *v = weighted<T>(*v, tb.wv[x >> 3]);
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) p[j] = 0u;
                if (i == 0) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4 *>(drow + ((((cg & 1) * 4 + j) ^ (s & 7)) << 4)) = zero8();
                }
            }
            tmem_st16(tl + cg * 16, p);
            if constexpr (DG) {
                rowsum[cg][s] = of_row + (first ? 0.f : rowsum[cg][s]);
                colsum[quad][cg * 32 + lane] = of_column + (first ? 0.f : colsum[quad][cg * 32 + lane]);
            }
            fence_async_smem();
            tmem_st_wait();
        }
        tc_fence_before();
        ok = __syncthreads_and(ok);
        if (!ok) break;
        if (i > 0 && i + 1 < nv) {                               // the tile before has left its buffers
            if (tid == 32) load_v(i + 1, h1, pb1);
            ++loads_v;
        }
        if (warp == kIssue && elect_one()) {
            ok = mbar_wait(&bar_s, i & 1);
            if (ok) {
                tc_fence_after();
                constexpr uint32_t narrow = instr_desc(AbFmt<T>::v, false, true, kP), wide = instr_desc(AbFmt<T>::v, false, false, NT);
                const uint32_t q0 = smem_u32(smQ), k0 = smem_u32(smK);
                const uint32_t v_ = smem_u32(sV), d_ = smem_u32(sD), e_ = smem_u32(smE), s_ = smem_u32(smS), g_ = smem_u32(smG);
#pragma unroll 1
                for (int kk = 0; kk < kQ / 16; ++kk)             // dv from the chunk, from the future; S^T q
                    umma_tmem(tmem + cOwn, tmem + kk * 8, smem_desc(d_ + kk * 2048, kSlab, 1024), narrow, kk > 0 ? 1u : 0u);
#pragma unroll 1
                for (int kk = 0; kk < NT / 16; ++kk)
                    umma(tmem + cFar, smem_desc(k0 + kk / 4 * kSlab + kk % 4 * 32, 16, 1024), smem_desc(g_ + kk * 2048, NT * 128, 1024), narrow, kk > 0 ? 1u : 0u);
#pragma unroll 1
                for (int kk = 0; kk < (DG ? NT / 16 : 0); ++kk)
                    umma(tmem + cOut, smem_desc(q0 + kk / 4 * kSlab + kk % 4 * 32, 16, 1024), smem_desc(s_ + kk * 2048, NT * 128, 1024), narrow, kk > 0 ? 1u : 0u);
#pragma unroll 1
                for (int kk = 0; kk < 4; ++kk) {                 // dq from the past, dk from the future
                    umma(tmem + cQ, smem_desc(e_ + kk * 32, 16, 1024), smem_desc(s_ + kk * 32, 16, 1024), wide, i > 0 || kk > 0 ? 1u : 0u);
                    umma(tmem + cK, smem_desc(v_ + kk * 32, 16, 1024), smem_desc(g_ + kk * 32, 16, 1024), wide, i > 0 || kk > 0 ? 1u : 0u);
                }
                umma_commit(&done_a);
            }
        }
        if (warp == kTables && i + 1 < nv && last) {             // the next head's, under the products; the turn before has been read
            Decays d;
            d.load(a.h, sg.batch, sg.t0, len, h1, lane);
            table(tables[(h1 - h0) & 1], d);
        }
        float whole = 0.f, among[4] = {};
        if constexpr (DG) {
            if (last && warp == kSums) {                         // a token's pairs: read here, behind the next barrier they may be another head's
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4 v = *reinterpret_cast<const float4 *>(&colsum[j][lane * 4]), w = *reinterpret_cast<const float4 *>(&rowsum[j][lane * 4]);
                    among[0] += v.x - w.x; among[1] += v.y - w.y; among[2] += v.z - w.z; among[3] += v.w - w.w;
                }
            }
            if (ok) ok = mbar_wait(&bar_s, i & 1);
            if (first) through = 0.f;
            if (ok)
                for (int q = tid; q < NT * 8; q += kT) {
                    const uint4 e = *reinterpret_cast<const uint4 *>(smS + q * 16), f = *reinterpret_cast<const uint4 *>(smG + q * 16);
                    vec::f2 v = vec::mul2(vec::widen<T>(e.x), vec::widen<T>(f.x));
                    v = vec::fma2(vec::widen<T>(e.y), vec::widen<T>(f.y), v);
                    v = vec::fma2(vec::widen<T>(e.z), vec::widen<T>(f.z), v);
                    through += both(vec::fma2(vec::widen<T>(e.w), vec::widen<T>(f.w), v));
                }
            whole = tb.whole[0];                         // read here: behind the next barrier its table may be another head's
            if (last) {
                float v = through;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                if (lane == 0) cross[warp] = v;
            }
        }
        if (ok) ok = mbar_wait(&done_a, i & 1);
        tc_fence_after();
        if (ok) {                                                // row s (or t), columns 16 cg ... of v's 64
            float own[16], far[16], o[16];
            vec::f2 f = vec::pack(0.f, 0.f), p = f, none = f;
            tmem_ld16(tl + cOwn + cg * 16, own);
            tmem_ld16(tl + cFar + cg * 16, far);
            if constexpr (DG) tmem_ld16(tl + cOut + cg * 16, o);
            const vec::f2 w = vec::pack(tb.ws[s], tb.ws[s]);
#pragma unroll
            for (int j = 0; j < 16; j += 8) {
                const int at = s * 128 + (((cg * 2 + j / 8) ^ (s & 7)) << 4);
                const uint4 v = *reinterpret_cast<const uint4 *>(sV + at), d = *reinterpret_cast<const uint4 *>(smE + at);
                const uint32_t vs[4] = {v.x, v.y, v.z, v.w}, ds[4] = {d.x, d.y, d.z, d.w};
                uint32_t to[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const vec::f2 far2 = vec::pack(far[j + 2 * k], far[j + 2 * k + 1]);
                    if constexpr (DG) {
                        f = vec::fma2(vec::widen<T>(vs[k]), far2, f);
                        p = vec::fma2(vec::widen<T>(ds[k]), vec::pack(o[j + 2 * k], o[j + 2 * k + 1]), p);
                    }
                    const vec::f2 sum = vec::fma2(w, far2, vec::pack(own[j + 2 * k], own[j + 2 * k + 1]));
                    if constexpr (kNarrow) none = vec::fma2(sum, vec::pack(0.f, 0.f), none);
                    to[k] = vec::narrow<T>(sum);
                }
                *reinterpret_cast<uint4 *>(sV + at) = make_uint4(to[0], to[1], to[2], to[3]);   // dv, where this thread alone has read v
            }
            if (kNarrow && both(none) != 0.f && s < len) uni::do_again(a.again, sg.seq, h, R);
            if constexpr (DG) {
                future[cg][s] = both(f) + (first ? 0.f : future[cg][s]);
                past[cg][s] = both(p) + (first ? 0.f : past[cg][s]);
            }
        }
        tc_fence_before();
        ok = __syncthreads_and(ok);
        if (!ok) break;
        if (i + 1 < nv) {
            if (tid == 32) load_s(h1, pb1);
            ++loads_s;
        }
        if (DG && last && warp == kSums) {
            float all = lane < 16 ? cross[lane] : 0.f, x[4] = {among[0], among[1], among[2], among[3]}, b[4] = {};
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
            all *= ex2_approx(whole);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 u = *reinterpret_cast<const float4 *>(&past[j][lane * 4]), z = *reinterpret_cast<const float4 *>(&future[j][lane * 4]);
                x[0] += u.x; x[1] += u.y; x[2] += u.z; x[3] += u.w;
                b[0] += z.x; b[1] += z.y; b[2] += z.z; b[3] += z.w;
            }
            // sums of x from each token on, of b before each
            float xs = x[0] + x[1] + x[2] + x[3], bs = b[0] + b[1] + b[2] + b[3];
            const float own_b = bs;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const float u = __shfl_down_sync(0xffffffffu, xs, o), v = __shfl_up_sync(0xffffffffu, bs, o);
                if (lane + o < 32) xs += u;
                if (lane >= o) bs += v;
            }
            bs -= own_b;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int t = lane * 4 + k;
                if (t < len) st_any(a.dg, a.dg_dtype, (token + t) * a.h.H + h, all + xs + bs);
                xs -= x[k];
                bs += b[k];
            }
        }
        h = h1;
        pb = pb1;
    }
    if (ok && warp == kIssue && elect_one()) from_chunk();
    if (ok) put_dv(nv - 1, h0 + (nv - 1) / a.h.PB, (nv - 1) % a.h.PB);
    if (ok) ok = mbar_wait(&done_b, (nv - 1) & 1);
    tc_fence_after();
    ok = __syncthreads_and(ok);
    if (ok) {                                                    // dq and dk: rows s (or t), NT / 4 columns a thread
        constexpr int kCols = NT / 4;
#pragma unroll
        for (int what = 0; what < 2; ++what) {
            const uint32_t at = tl + (what ? cK : cQ) + cg * kCols;
            uint8_t *to = what ? smN : smV;
#pragma unroll
            for (int j0 = 0; j0 < kCols; j0 += 16) {
                float x[16];
                tmem_ld16(at + j0, x);
                const int n = cg * kCols + j0;
                if constexpr (kNarrow) {
                    float none = 0.f;
#pragma unroll
                    for (int j = 0; j < 16; ++j) none = fmaf(x[j], 0.f, none);
                    if (none != 0.f && s < len) uni::do_again(a.again, sg.seq, h0, R);
                }
                if (a.parts > 1) {
                    float *o = a.part + (((long long)(what * a.parts + part) * a.tokens + token + s) * a.h.hk + m) * a.h.N + n;
#pragma unroll
                    for (int j = 0; j < 16; j += 4)
                        if (s < len && n + j < a.h.N) *reinterpret_cast<float4 *>(o + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
                } else {
#pragma unroll
                    for (int j = 0; j < 16; j += 8) {
                        const float e[8] = {x[j], x[j + 1], x[j + 2], x[j + 3], x[j + 4], x[j + 5], x[j + 6], x[j + 7]};
                        *reinterpret_cast<uint4 *>(to + (n + j) / 64 * kSlab + s * 128 + ((((n + j) % 64 / 8) ^ (s & 7)) << 4)) = pack8<T>(e);
                    }
                }
            }
        }
        __syncthreads();
        if (a.parts == 1) {
            const int pieces = a.h.N / 8;
            for (int x = tid; x < 2 * kQ * (NT / 8); x += kT) {
                const int what = x / (kQ * (NT / 8)), r = x / (NT / 8) % kQ, j = x % (NT / 8);
                if (r < len && j < pieces)
                    *reinterpret_cast<uint4 *>(static_cast<T *>(what ? a.dk : a.dq) + ((token + r) * a.h.hk + m) * a.h.N + j * 8) =
                        *reinterpret_cast<const uint4 *>((what ? smN : smV) + j / 8 * kSlab + r * 128 + (((j & 7) ^ (r & 7)) << 4));
            }
        }
    } else if (tid == 0) {
        atomicExch(a.status, kErrDecay + 3);
    }
    if (!ok && warp == kIssue && elect_one()) {                  // leave nothing in flight
        drain_mmas(&unused);
        drain_loads(&bar_qk, 1, 1);
        drain_loads(bar_v, 2, loads_v);
        drain_loads(&bar_s, 1, loads_s);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem, 512);
}

// dq and dk of chunks whose heads were walked by several blocks: their parts added up in order.
template <class T> __global__ void __launch_bounds__(256) decay_sum_parts(const float *part, int parts, long long each, T *dq, T *dk) {
    pdl_begin();
    const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= 2 * each) return;
    const int what = i >= each;
    const float *p = part + what * parts * each + (i - what * each);
    float4 v = *reinterpret_cast<const float4 *>(p);
    for (int k = 1; k < parts; ++k) {
        const float4 u = *reinterpret_cast<const float4 *>(p + k * each);
        v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
    }
    uint2 o;
    o.x = pack2<T>(v.x, v.y);
    o.y = pack2<T>(v.z, v.w);
    *reinterpret_cast<uint2 *>((what ? dk : dq) + (i - what * each)) = o;
}

}  // namespace unitc
}  // namespace bissd
