// The causal decay attention on the tensor cores (bf16), in chunks of 128 tokens.  With c_t the sum of the chunk's log decays up to
// and with token t, and S the state that enters the chunk,
//     o_t = scale [ e^{c_t} S^T q_t + sum_{s <= t} e^{c_t - c_s} (q_t.k_s) v_s ],    S' = e^{c_end} S + sum_s k_s (e^{c_end - c_s} v_s)^T
// so a chunk is four products of 128 rows; only S' waits for the chunk before it.
//   decay_states   walks the chunks of one head with S in registers and writes what enters each: the k v^T products alone
//   decay_chunks   all chunks at once, given the states
// Heads of v are taken 64 columns at a time: with the same weights, v's parts are heads of their own that share q, k and g.  Head sizes
// that fill no tile are completed by the loads with zeros.  Log decays count in powers of two and no lower than 2^-200 a token, which
// fp32 has no number for: -inf never meets +inf.  Factors that reach to a chunk's ends are 2 to the power of a sum that starts there,
// so that a strong decay elsewhere in the chunk costs them no digits.
#pragma once
#include "tc_tma.cuh"
#include "uni_plan.cuh"

namespace bissd {
namespace unitc {

using namespace tc;
using uni::Plan;
using uni::Segment;
typedef __nv_bfloat16 bf16;

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
    __device__ __forceinline__ void log2(const Heads &a) {       // bf16 or fp32
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = fmaxf(__uint_as_float(a.g_dtype == BISSD_F32 ? raw[i] : raw[i] << 16) * 1.44269504f, -200.f);
    }
    // Sums up to and with each token.
    __device__ __forceinline__ void prefix(float (&c)[4], int lane) const {
        c[0] = v[0];
#pragma unroll
        for (int i = 1; i < 4; ++i) c[i] = c[i - 1] + v[i];
        float mine = c[3], sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const float u = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += u;
        }
        const float before = __shfl_up_sync(0xffffffffu, sum, 1);
        if (lane > 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] += before;
        }
    }
    // Sums of the tokens behind each.
    __device__ __forceinline__ void suffix(float (&c)[4], int lane) const {
        c[3] = 0.f;
#pragma unroll
        for (int i = 2; i >= 0; --i) c[i] = c[i + 1] + v[i + 1];
        float sum = c[0] + v[0];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const float u = __shfl_down_sync(0xffffffffu, sum, o);
            if (lane + o < 32) sum += u;
        }
        const float behind = __shfl_down_sync(0xffffffffu, sum, 1);
        if (lane < 31) {
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] += behind;
        }
    }
};

// Rows of a tile behind the sequence's end: a packed neighbour's, of whatever values, become zeros.
__device__ __forceinline__ void clear_rows(uint8_t *slab, int from, int tid, int threads) {
    for (int i = from * 8 + tid; i < kQ * 8; i += threads) *reinterpret_cast<uint4 *>(slab + i * 16) = zero8();
}

// ---- the states that enter the chunks ------------------------------------------------------------------------------------
// Forwards S' as above; backwards (v the outputs' gradient, k the queries) the gradient that enters each chunk from its right,
// G' = e^{c_end} G + sum_t q_t (scale e^{c_t} do_t)^T.  A block walks the chunks of one (segment, head, 64 columns), S or G in
// registers (a row n and 32 columns a thread) and the next chunk's rows on their way; v's rows are weighted in place.
// exact: the weighted row is given to the tensor cores in three bf16 parts, each what is left of those before, so that the states
// that leave the library are fp32's.  The tiles that the other kernels read are bf16 in any case: they meet bf16 factors.
struct StatesParams {
    Heads h;
    Plan seg, chunk;
    int reverse, exact, by_seq;                                  // by_seq: init and fin hold a state a sequence, not a segment
    const float *init;
    float *fin, *decay;                                          // decay: (segments, H) the segment's whole decay, or NULL
    bf16 *tiles;                                                 // (chunks, H, PB, NT, 64), or NULL
    int *status;
};
inline size_t states_smem(int NT) { return 1024 + 2 * (size_t)(NT / 64) * kSlab + 2 * (size_t)kSlab; }

template <int NT> __global__ void __launch_bounds__(256, 2)
decay_states(StatesParams a, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV) {
    pdl_begin();
    constexpr int kSlabs = NT / 64;
    extern __shared__ uint8_t dyn[];
    __shared__ uint64_t full[2], done, unused;
    __shared__ uint32_t tmem_slot;
    __shared__ float w[3][kQ], whole[3];                          // of three steps: a warp may be one behind another
    uint8_t *smK = smem_align1024(dyn), *smV = smK + 2 * kSlabs * kSlab;   // two stages of each
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int pb = blockIdx.x % a.h.PB, h = blockIdx.x / a.h.PB % a.h.H, si = blockIdx.x / (a.h.PB * a.h.H), hq = h * a.h.hk / a.h.H;
    const Segment s = uni::segment(a.seg, si);
    if (s.len == 0) return;                                      // packed: fewer segments than there could be
    const int nc = ceil_div(s.len, kQ), c0 = uni::segments(a.chunk, s.seq).x + s.idx * (a.seg.seg / kQ);
    auto place = [&](int i) { return a.reverse ? nc - 1 - i : i; };        // chunk of the segment at step i
    auto load = [&](int i) {
        const int st = i & 1, t = s.t0 + place(i) * kQ;
        mbar_expect_tx(&full[st], (kSlabs + 1) * kSlab);
        for (int j = 0; j < kSlabs; ++j) tma_load4(smK + (st * kSlabs + j) * kSlab, &tmK, j * 64, hq, t, s.batch, &full[st]);
        tma_load4(smV + st * kSlab, &tmV, pb * kP, h, t, s.batch, &full[st]);
    };
    auto weights = [&](int i, Decays d) {                        // one warp
        const int len = min(kQ, s.len - place(i) * kQ);
        float c[4], p[4];
        d.log2(a.h);
        d.prefix(p, lane);
        if (a.reverse) {
#pragma unroll
            for (int k = 0; k < 4; ++k) c[k] = p[k] + a.h.log_scale;
        } else {
            d.suffix(c, lane);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) w[i % 3][lane * 4 + k] = lane * 4 + k < len ? exp2f(c[k]) : 0.f;
        if (lane == 31) whole[i % 3] = p[3];
    };
    if (warp == 0) tmem_alloc(&tmem_slot, 64);
    if (tid == 32) {
        mbar_init(&full[0], 1);
        mbar_init(&full[1], 1);
        mbar_init(&done, 1);
        fence_mbar_init();
        load(0);
    }
    Decays next;                                                 // warp 2: of the step after the one whose weights it writes
    auto fetch = [&](int i) {
        if (i < nc) next.load(a.h, s.batch, s.t0 + place(i) * kQ, min(kQ, s.len - place(i) * kQ), h, lane);
    };
    if (warp == 2) {
        fetch(0);
        weights(0, next);
        fetch(1);
    }
    const int n = (warp & 3) * 32 + lane, half = warp >> 2, col = pb * kP + half * 32;
    const long long at = (((long long)(a.by_seq ? s.seq : si) * a.h.H + h) * a.h.N + n) * a.h.P + col;
    float S[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) S[j] = a.init && n < a.h.N && col + j < a.h.P ? a.init[at + j] : 0.f;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    constexpr uint32_t idesc = instr_desc(1, true, true, kP);
    bool ok = true;
    int loads = 1, waits = 0;                                    // loads asked for, uses of `done`
    float total = 0.f;
    for (int i = 0; i < nc; ++i) {
        const int st = i & 1, len = min(kQ, s.len - place(i) * kQ);
        if (i + 1 < nc) {                                        // the stage was read by the MMAs of the step before, which are done
            if (tid == 32) load(i + 1);
            ++loads;
        }
        ok = ok && mbar_wait(&full[st], (i >> 1) & 1);
        uint8_t *v = smV + st * kSlab;
        uint4 rows[4];                                           // v's as loaded
        auto weigh = [&](int part) {                             // part 0, 1 or 2 of the weighted rows to where v's were
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int x = tid + k * 256, row = x >> 3;
                const float f = row < len ? w[i % 3][row] : 0.f;
                float e[8], r[8];
                unpack8<bf16>(rows[k], e);
#pragma unroll
                for (int m = 0; m < 8; ++m) e[m] = row < len ? e[m] * f : 0.f;
                uint4 out = pack8<bf16>(e);
                for (int q = 0; q < part; ++q) {
                    unpack8<bf16>(out, r);
#pragma unroll
                    for (int m = 0; m < 8; ++m) e[m] -= r[m];
                    out = pack8<bf16>(e);
                }
                *reinterpret_cast<uint4 *>(v + x * 16) = out;
            }
            fence_async_smem();
        };
        if (ok) {
            if (a.seg.packed && len < kQ)
                for (int j = 0; j < kSlabs; ++j) clear_rows(smK + (st * kSlabs + j) * kSlab, len, tid, 256);
#pragma unroll
            for (int k = 0; k < 4; ++k) rows[k] = *reinterpret_cast<const uint4 *>(v + (tid + k * 256) * 16);
            weigh(0);
        }
        if (warp == 2 && i + 1 < nc) {
            weights(i + 1, next);
            fetch(i + 2);
        }
        tc_fence_before();                                       // the last step's loads from tensor memory
        ok = __syncthreads_and(ok);
        if (!ok) break;
        auto issue = [&](uint32_t first) {
            tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < kQ / 16; ++kk)                 // where NT is 64, rows 64 ... 127 are v's columns: products of no use
                umma(tmem, smem_desc(smem_u32(smK + st * kSlabs * kSlab) + kk * 2048, NT == 64 ? 2 * kSlab : kSlab, 1024),
                     smem_desc(smem_u32(v) + kk * 2048, kSlab, 1024), idesc, kk > 0 ? 1u : first);
            umma_commit(&done);
        };
        if (warp == 0 && elect_one()) issue(0u);
        if (a.tiles && n < NT) {                                 // what enters this chunk
            uint4 *o = reinterpret_cast<uint4 *>(a.tiles + ((((long long)(c0 + place(i)) * a.h.H + h) * a.h.PB + pb) * NT + n) * kP + half * 32);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float e[8] = {S[8 * j], S[8 * j + 1], S[8 * j + 2], S[8 * j + 3], S[8 * j + 4], S[8 * j + 5], S[8 * j + 6], S[8 * j + 7]};
                o[j] = pack8<bf16>(e);
            }
        }
        ok = mbar_wait(&done, waits & 1);
        ++waits;
        if (a.exact) {
#pragma unroll
            for (int part = 1; part < 3; ++part) {
                if (ok) weigh(part);
                ok = __syncthreads_and(ok);
                if (ok && warp == 0 && elect_one()) issue(1u);
                if (ok) ok = mbar_wait(&done, waits & 1);
                ++waits;
            }
        }
        if (!ok) continue;                                       // leaves at the next barrier
        tc_fence_after();
        const float d = exp2f(whole[i % 3]);
        total += whole[i % 3];
        float v32[32];
        tmem_ld32(tmem_lane_base(tmem) + half * 32, v32);
#pragma unroll
        for (int j = 0; j < 32; ++j) S[j] = fmaf(S[j], d, v32[j]);
    }
    ok = __syncthreads_and(ok);
    if (ok) {
        if (a.fin && n < a.h.N) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (col + j < a.h.P) a.fin[at + j] = S[j];
        }
        if (a.decay && pb == 0 && tid == 0) a.decay[(long long)si * a.h.H + h] = exp2f(total);
    } else if (tid == 0) {
        atomicExch(a.status, kErrDecay + 1);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        if (!ok && elect_one()) {                                // leave nothing in flight
            drain_mmas(&unused);
            drain_loads(full, 2, loads);
        }
        __syncwarp();
        tmem_dealloc(tmem, 64);
    }
}

// ---- the outputs -----------------------------------------------------------------------------------------------------
// A block has one chunk of one head of q and k, and walks `vpc` of the tiles of v that share them: Q, K and their product stay, in
// shared and tensor memory, and per tile come v's rows and the state.  The product, weighted by the decays and rounded to bf16 (it
// meets v's bf16), takes K's place in shared memory.  Where a whole block of 64 x 64 lies below the diagonal, the weight is a row
// factor times a column factor, both counted from the block's corner and at most 1; on the diagonal it is one 2^x an element.
// Two blocks an SM: one's loads and element-wise work run under the other's MMAs.
struct ChunksParams {
    Heads h;
    Plan chunk;
    int vpc, parts;                                              // tiles of v a block, blocks a (chunk, head of q)
    int tiles_rows;                                              // NT
    bf16 *o;                                                     // (tokens, H, P) contiguous
    int *status;
};
inline size_t chunks_smem(int NT) { return 1024 + (size_t)(NT / 64) * kSlab + 2 * (size_t)kSlab + (size_t)kSlab + (size_t)NT * 128; }

template <int NT> __global__ void __launch_bounds__(256, 2)
decay_chunks(ChunksParams a, const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
             const __grid_constant__ CUtensorMap tmS) {
    pdl_begin();
    constexpr int kSlabs = NT / 64;
    extern __shared__ uint8_t dyn[];
    __shared__ uint64_t bar_qk, bar_v, done, unused;
    __shared__ uint32_t tmem_slot;
    __shared__ __align__(16) float cs[2][kQ], below[2][64];      // c_t; 2^(c_63 - c_s) of the first 64 tokens
    uint8_t *smQ = smem_align1024(dyn), *smK = smQ + kSlabs * kSlab, *smV = smK + 2 * kSlab, *smS = smV + kSlab;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int part = blockIdx.x % a.parts, m = blockIdx.x / a.parts % a.h.hk, ci = blockIdx.x / (a.parts * a.h.hk);
    const Segment s = uni::segment(a.chunk, ci);
    if (s.len == 0) return;
    const int R = a.h.H / a.h.hk, v0 = part * a.vpc, nv = min(a.vpc, R * a.h.PB - v0);
    auto head = [&](int i) { return m * R + (v0 + i) / a.h.PB; };
    auto load_v = [&](int i) {
        const int h = head(i), pb = (v0 + i) % a.h.PB;
        mbar_expect_tx(&bar_v, kSlab + NT * 128);
        tma_load4(smV, &tmV, pb * kP, h, s.t0, s.batch, &bar_v);
        tma_load2(smS, &tmS, 0, ((ci * a.h.H + h) * a.h.PB + pb) * NT, &bar_v);
    };
    auto table = [&](int i, Decays d) {                          // one warp
        float c[4];
        d.log2(a.h);
        d.prefix(c, lane);
        const float corner = __shfl_sync(0xffffffffu, c[3], 15);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            cs[i & 1][lane * 4 + k] = c[k];
            if (lane < 16) below[i & 1][lane * 4 + k] = exp2f(corner - c[k]);
        }
    };
    if (warp == 0) tmem_alloc(&tmem_slot, 256);
    if (tid == 32) {
        mbar_init(&bar_qk, 1);
        mbar_init(&bar_v, 1);
        mbar_init(&done, 1);
        fence_mbar_init();
        mbar_expect_tx(&bar_qk, 2 * kSlabs * kSlab);
        for (int j = 0; j < kSlabs; ++j) {
            tma_load4(smQ + j * kSlab, &tmQ, j * 64, m, s.t0, s.batch, &bar_qk);
            tma_load4(smK + j * kSlab, &tmK, j * 64, m, s.t0, s.batch, &bar_qk);
        }
        load_v(0);
    }
    Decays next;                                                 // warp 2: of the next head
    auto fetch = [&](int i) {
        if (i < nv && head(i) != head(i - 1)) next.load(a.h, s.batch, s.t0, s.len, head(i), lane);
    };
    if (warp == 2) {
        next.load(a.h, s.batch, s.t0, s.len, head(0), lane);
        table(0, next);
        fetch(1);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot, tl = tmem_lane_base(tmem);  // columns: 0 q.k, 128 inside the chunk, 192 from the state
    int loads = 1, waits = 0;
    bool ok = true;
    if (warp == 0 && elect_one()) {
        ok = mbar_wait(&bar_qk, 0);
        if (ok) {
            constexpr uint32_t idesc = instr_desc(1, false, false, kQ);
#pragma unroll
            for (int kk = 0; kk < NT / 16; ++kk)
                umma(tmem, smem_desc(smem_u32(smQ + kk / 4 * kSlab) + kk % 4 * 32, 16, 1024),
                     smem_desc(smem_u32(smK + kk / 4 * kSlab) + kk % 4 * 32, 16, 1024), idesc, kk > 0 ? 1u : 0u);
            umma_commit(&done);
        }
    }
    if (ok) ok = mbar_wait(&done, 0);
    ++waits;
    const int t = (warp & 3) * 32 + lane, half = warp >> 2;      // this thread: row t, columns of `half` of each tile
    const bool diagonal = (t >> 6) == half, empty = (t >> 6) < half;
    for (int i = 0; i < nv; ++i) {
        if (ok) ok = mbar_wait(&bar_v, i & 1);
        if (ok && a.chunk.packed && s.len < kQ) {
            clear_rows(smV, s.len, tid, 256);
            fence_async_smem();
        }
        ok = __syncthreads_and(ok);
        if (!ok) break;
        tc_fence_after();
        if (warp == 0 && elect_one()) {                          // from the state: Q S
            constexpr uint32_t idesc = instr_desc(1, false, true, kP);
#pragma unroll
            for (int kk = 0; kk < NT / 16; ++kk)
                umma(tmem + 192, smem_desc(smem_u32(smQ + kk / 4 * kSlab) + kk % 4 * 32, 16, 1024),
                     smem_desc(smem_u32(smS) + kk * 2048, NT * 128, 1024), idesc, kk > 0 ? 1u : 0u);
        }
        const float *c = cs[i & 1];
        const float ct = c[t] + a.h.log_scale;
        uint8_t *row = smK + half * kSlab + t * 128;             // 64 weighted pairs, 16-byte pieces swizzled
        if (empty) {
            if (i == 0) {
#pragma unroll
                for (int j = 0; j < 8; ++j) *reinterpret_cast<uint4 *>(row + ((j ^ (t & 7)) << 4)) = zero8();
            }
        } else {
            const float rt = exp2f(ct - c[63]);
#pragma unroll
            for (int j0 = 0; j0 < 64; j0 += 32) {
                float x[32];
                tmem_ld32(tl + half * 64 + j0, x);
#pragma unroll
                for (int j = 0; j < 32; j += 4) {
                    const int col = j0 + j;
                    if (diagonal) {
                        const float4 f = *reinterpret_cast<const float4 *>(c + half * 64 + col);
                        const int td = t & 63;
                        x[j] = col <= td ? x[j] * ex2_approx(ct - f.x) : 0.f;
                        x[j + 1] = col + 1 <= td ? x[j + 1] * ex2_approx(ct - f.y) : 0.f;
                        x[j + 2] = col + 2 <= td ? x[j + 2] * ex2_approx(ct - f.z) : 0.f;
                        x[j + 3] = col + 3 <= td ? x[j + 3] * ex2_approx(ct - f.w) : 0.f;
                    } else {
                        const float4 f = *reinterpret_cast<const float4 *>(below[i & 1] + col);
                        x[j] *= rt * f.x;
                        x[j + 1] *= rt * f.y;
                        x[j + 2] *= rt * f.z;
                        x[j + 3] *= rt * f.w;
                    }
                }
#pragma unroll
                for (int j = 0; j < 32; j += 8) {
                    const float e[8] = {x[j], x[j + 1], x[j + 2], x[j + 3], x[j + 4], x[j + 5], x[j + 6], x[j + 7]};
                    *reinterpret_cast<uint4 *>(row + ((((j0 + j) >> 3) ^ (t & 7)) << 4)) = pack8<bf16>(e);
                }
            }
        }
        fence_async_smem();
        __syncthreads();
        if (warp == 0 && elect_one()) {                          // inside the chunk: the weighted pairs times v
            constexpr uint32_t idesc = instr_desc(1, false, true, kP);
#pragma unroll
            for (int kk = 0; kk < kQ / 16; ++kk)
                umma(tmem + 128, smem_desc(smem_u32(smK + kk / 4 * kSlab) + kk % 4 * 32, 16, 1024),
                     smem_desc(smem_u32(smV) + kk * 2048, kSlab, 1024), idesc, kk > 0 ? 1u : 0u);
            umma_commit(&done);
        }
        const bool another = i + 1 < nv && head(i + 1) != head(i);
        if (warp == 2 && i + 1 < nv) {
            if (another) {
                table(i + 1, next);
            } else {
                for (int k = lane; k < kQ; k += 32) cs[(i + 1) & 1][k] = c[k];
                for (int k = lane; k < 64; k += 32) below[(i + 1) & 1][k] = below[i & 1][k];
            }
            fetch(i + 2);
        }
        ok = mbar_wait(&done, waits & 1);
        ++waits;
        ok = __syncthreads_and(ok);
        if (!ok) break;
        tc_fence_after();
        if (i + 1 < nv) {
            if (tid == 32) load_v(i + 1);
            ++loads;
        }
        // o = inside + scale e^{c_t} from the state; whole rows leave through the first slab of the weighted pairs
        {
            const float f = exp2f(ct);
            float x[32], y[32];
            tmem_ld32(tl + 128 + half * 32, x);
            tmem_ld32(tl + 192 + half * 32, y);
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
                float e[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) e[k] = fmaf(y[j + k], f, x[j + k]);
                *reinterpret_cast<uint4 *>(smK + t * 128 + (((half * 4 + (j >> 3)) ^ (t & 7)) << 4)) = pack8<bf16>(e);
            }
        }
        tc_fence_before();
        __syncthreads();
        const int h = head(i), col = (v0 + i) % a.h.PB * kP + (tid & 7) * 8;
        if (col < a.h.P) {
            bf16 *o = a.o + ((long long)s.batch * a.chunk.L + s.t0) * a.h.H * a.h.P + (long long)h * a.h.P + col;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int r = (tid >> 3) + k * 32;
                if (r < s.len) *reinterpret_cast<uint4 *>(o + (long long)r * a.h.H * a.h.P) = *reinterpret_cast<const uint4 *>(smK + r * 128 + (((tid & 7) ^ (r & 7)) << 4));
            }
        }
    }
    ok = __syncthreads_and(ok);
    if (!ok && tid == 0) atomicExch(a.status, kErrDecay + 2);
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        if (!ok && elect_one()) {                                // leave nothing in flight
            drain_mmas(&unused);
            drain_loads(&bar_qk, 1, 1);
            drain_loads(&bar_v, 1, loads);
        }
        __syncwarp();
        tmem_dealloc(tmem, 256);
    }
}

}  // namespace unitc
}  // namespace bissd
