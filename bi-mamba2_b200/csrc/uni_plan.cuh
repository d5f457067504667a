// Where the sequences of a decay attention call lie, and the segments that their tokens are dealt out in.  A batch's rows are
// sequences of one length, and a segment's place is arithmetic; packed sequences have theirs on the device, so a small
// kernel writes a table of their segments, and a launch has as many blocks as there can be at most.
#pragma once
#include "common.cuh"

namespace bissd {
namespace uni {

struct Plan {
    int packed, L, seg, per_seq, most;                           // most: segments there can be (all of them where not packed)
    const int4 *table;                                           // packed: first token, tokens, sequence, 2 * index + last
    const int *first;                                            // packed: (nseq + 1) first segment of each sequence
    const int *bounds;                                           // packed, each sequence one segment: (nseq + 1) boundaries, no table; or NULL
};
struct Segment {
    int batch, t0, len, seq, idx;                                // len 0: there is no such segment
    bool last;
};

__device__ __forceinline__ Segment segment(const Plan &p, int i) {
    Segment s;
    if (p.packed) {
        const int4 e = __ldg(p.table + i);
        s.batch = 0; s.t0 = e.x; s.len = e.y; s.seq = e.z; s.idx = e.w >> 1; s.last = e.w & 1;
    } else {
        s.batch = s.seq = i / p.per_seq;
        s.idx = i % p.per_seq;
        s.t0 = s.idx * p.seg;
        s.len = min(p.seg, p.L - s.t0);
        s.last = s.idx == p.per_seq - 1;
    }
    return s;
}
// The same where a plan may have bounds.
__device__ __forceinline__ Segment segment_or_sequence(const Plan &p, int i) {
    if (!p.bounds) return segment(p, i);
    Segment s;
    s.batch = s.idx = 0; s.t0 = p.bounds[i]; s.len = p.bounds[i + 1] - s.t0; s.seq = i; s.last = true;
    return s;
}
// The segments of a sequence: first and how many.
__device__ __forceinline__ int2 segments(const Plan &p, int seq) {
    if (!p.packed) return make_int2(seq * p.per_seq, p.per_seq);
    return make_int2(p.first[seq], p.first[seq + 1] - p.first[seq]);
}

// Calls in fp16 on the tensor cores whose products leave the type's range somewhere: heads of sequences that are to be done again, on CUDA
// cores in fp32.  flags[0]: any of them; flags[1 + sequence H + head].  Cleared in a call's first kernel that goes by sequences, set in later
// ones, read in those behind; `bad`: by blocks of decay_states, whether the state that leaves the library left the range.
struct Again {
    int *flags, *bad;
    int H, bads, per_segment;                                    // bads: blocks, per_segment of them to a segment of `seg`
    Plan seg;
};
__device__ __forceinline__ bool again(const int *flags, int H, int seq, int h) { return flags[0] && flags[1 + (long long)seq * H + h]; }
// Every gradient of heads that share q and k is done again where one of them is: R heads, R = 1 for outputs.
__device__ __forceinline__ void do_again(const Again &a, int seq, int h, int R) {
    a.flags[0] = 1;
    for (int r = 0; r < R; ++r) a.flags[1 + (long long)seq * a.H + h / R * R + r] = 1;
}
__device__ __forceinline__ void do_again_states(const Again &a, int R, int threads) {   // what decay_states found; all blocks of a launch
    for (long long i = (long long)blockIdx.x * threads + threadIdx.x; i < a.bads; i += (long long)gridDim.x * threads)
        if (a.bad[i]) do_again(a, segment(a.seg, (int)i / a.per_segment).seq, (int)i % a.per_segment / (a.per_segment / a.H), R);
}

struct PlanOut {                                                 // one table for each segment length
    int seg, most;
    int4 *table;
    int *first, *bounds;                                         // bounds (nseq + 1): the boundaries as taken
};

// Inclusive scan over a block of 1024 threads; `op` max or sum.
template <class F> __device__ __forceinline__ int block_scan(int v, int *warps, F op, int none) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v = op(v, u);
    }
    __syncthreads();
    if (lane == 31) warps[warp] = v;
    __syncthreads();
    int before = lane < warp ? warps[lane] : none;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) before = op(before, __shfl_xor_sync(0xffffffffu, before, o));
    return op(before, v);
}

// What packed sequences leave over.  Zeros in the rows of outputs that belong to no sequence, those before the first one and behind
// the last; and the states of sequences without a token, which stay as they were (start NULL: zeros).
struct RestParams {
    int L, nseq, outs;
    char *out[6];                                                // outputs and their rows' bytes, even
    long long bytes[6];
    float *parts;                                                // n_parts arrays of (L, part_row), or NULL
    int n_parts;
    long long part_row;
    const float *start;
    float *end;                                                  // (nseq, per), or NULL
    long long per;
    int *status;                                                 // cleared, or NULL
};
// One of `blocks` blocks' share; bounds: nseq + 1.
__device__ __forceinline__ void rest_of(const RestParams &a, const int *bounds, int block, int blocks) {
    const int head = bounds[0], tail = bounds[a.nseq], rows = head + a.L - tail;
    for (int i = block; i < rows; i += blocks) {
        const long long row = i < head ? i : tail + i - head;
        for (int o = 0; o < a.outs; ++o) {
            uint16_t *p = reinterpret_cast<uint16_t *>(a.out[o] + row * a.bytes[o]);
            for (long long e = threadIdx.x; e < a.bytes[o] / 2; e += blockDim.x) p[e] = 0;
        }
        for (int k = 0; k < a.n_parts; ++k)
            for (long long e = threadIdx.x; e < a.part_row; e += blockDim.x) a.parts[((long long)k * a.L + row) * a.part_row + e] = 0.f;
    }
    if (a.end)
        for (int s = block; s < a.nseq; s += blocks)
            if (bounds[s] == bounds[s + 1])
                for (long long e = threadIdx.x; e < a.per; e += blockDim.x) a.end[s * a.per + e] = a.start ? a.start[s * a.per + e] : 0.f;
}
__global__ void __launch_bounds__(1024) decay_rest(RestParams a, const int *bounds) {
    pdl_begin();
    rest_of(a, bounds, blockIdx.x, gridDim.x);
}

constexpr int kNear = 1024;                                      // sequences that one pass of a block's scan covers
// A block for each of `tables` tables, and up to kNear sequences blocks behind them for what these leave over: every block finds all
// boundaries, and a launch is saved.  Boundaries are taken to 0 ... L and never back, so every segment lies inside the tensors whatever
// the caller's array holds.
__global__ void __launch_bounds__(1024) decay_plan(const int *cu, int nseq, int L, PlanOut a, PlanOut b, int tables, RestParams rest) {
    pdl_begin();
    __shared__ int warps[32], carry[2], near_first[kNear + 1], near_bounds[kNear + 1];   // the search below is a chain of reads
    const bool plans = blockIdx.x < tables;
    const PlanOut o = blockIdx.x ? b : a;
    const int tid = threadIdx.x;
    auto most = [](int x, int y) { return max(x, y); };
    auto sum = [](int x, int y) { return x + y; };
    auto inside = [&](int i) { return max(0, min(cu[i], L)); };
    if (rest.status && blockIdx.x == 0 && tid == 0) *rest.status = 0;
    if (tid == 0) {
        carry[1] = near_first[0] = 0;
        carry[0] = near_bounds[0] = inside(0);
        if (plans) {
            o.first[0] = 0;
            o.bounds[0] = carry[0];
        }
    }
    __syncthreads();
    for (int s0 = 0; s0 < nseq; s0 += 1024) {
        const int s = s0 + tid;
        const int to = s < nseq ? inside(s + 1) : 0, from = s < nseq ? inside(s) : 0;
        const int end = max(carry[0], block_scan(to, warps, most, 0));
        const int start = max(carry[0], block_scan(from, warps, most, 0));
        const int upto = carry[1] + block_scan(s < nseq ? (end - start + o.seg - 1) / o.seg : 0, warps, sum, 0);
        if (s < nseq) {
            if (plans) {
                o.first[s + 1] = upto;
                o.bounds[s + 1] = end;
            }
            if (s < kNear) {
                near_first[s + 1] = upto;
                near_bounds[s + 1] = end;
            }
        }
        __syncthreads();
        if (tid == 1023) {
            carry[0] = end;
            carry[1] = upto;
        }
        __syncthreads();
    }
    if (!plans) {
        rest_of(rest, near_bounds, blockIdx.x - tables, gridDim.x - tables);
        return;
    }
    const int *first = nseq <= kNear ? near_first : o.first, *bounds = nseq <= kNear ? near_bounds : o.bounds;
    for (int i = tid; i < o.most; i += 1024) {
        int lo = 0, hi = nseq;                                   // the sequence that segment i belongs to: first[lo] <= i < first[lo + 1]
        if (i >= carry[1]) {
            o.table[i] = make_int4(0, 0, 0, 0);
            continue;
        }
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (first[mid] <= i) lo = mid;
            else hi = mid;
        }
        const int idx = i - first[lo], t0 = bounds[lo] + idx * o.seg;
        o.table[i] = make_int4(t0, min(o.seg, bounds[lo + 1] - t0), lo, 2 * idx + (t0 + o.seg >= bounds[lo + 1]));
    }
}

}  // namespace uni
}  // namespace bissd
