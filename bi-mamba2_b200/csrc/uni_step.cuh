// One token of every request through the causal decay attention, states updated in place:
//     S = e^g S + k v^T,   o = scale S^T q            (kdim x vdim, fp32, per request and head)
// Bound by the states' bytes: each is read once and written once, 8 bytes an element against 5 operations.  A block has
// 32 columns of one state, so nothing is summed across blocks; its eight warps take the rows in turn, 16 bytes a lane and
// every row of the block asked for before the first is used.  The products with q are summed over the lanes that share
// columns, then over the warps, in a fixed order.
#pragma once
#include "common.cuh"

namespace bissd {
namespace uni {

struct StepParams {
    View q, k, v, g;
    MutView o;
    float *state;
    long long slot_stride;
    const int *slots;
    int batch, H, hk, N, P, nslots, g_dtype, column_blocks;
    float scale;
};

constexpr int kStepThreads = 256, kStepColumns = 32;

// VEC columns a lane, PASSES rows a thread: kdim <= PASSES * (8 VEC).
template <class T, int VEC, int PASSES>
__global__ void __launch_bounds__(kStepThreads, VEC == 4 && PASSES <= 4 ? 6 : 2) decay_step(StepParams a) {
    pdl_begin();
    constexpr int kLanes = kStepColumns / VEC, kRows = kStepThreads / kLanes;
    __shared__ float part[kStepThreads / 32][kStepColumns];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int cb = blockIdx.x % a.column_blocks, h = blockIdx.x / a.column_blocks % a.H, i = blockIdx.x / (a.column_blocks * a.H);
    const int c = cb * kStepColumns + tid % kLanes * VEC, n0 = tid / kLanes, hq = h * a.hk / a.H;
    const int slot = a.slots ? a.slots[i] : i;
    const int oc = cb * kStepColumns + tid;                      // the column that this thread writes of o
    if (slot < 0 || slot >= a.nslots) {
        if (tid < kStepColumns && oc < a.P) st<T>(a.o.ptr, i * a.o.sb + h * a.o.sh + oc, 0.f);
        return;
    }
    float *base = a.state + slot * a.slot_stride + (long long)h * a.N * a.P + c;
    float s[PASSES][VEC];
#pragma unroll
    for (int r = 0; r < PASSES; ++r) {
        const int n = n0 + r * kRows;
        const bool in = n < a.N && c < a.P;
        if constexpr (VEC == 4) {
            const float4 f = in ? __ldcs(reinterpret_cast<const float4 *>(base + (long long)n * a.P)) : make_float4(0.f, 0.f, 0.f, 0.f);
            s[r][0] = f.x; s[r][1] = f.y; s[r][2] = f.z; s[r][3] = f.w;
        } else {
            s[r][0] = in ? base[(long long)n * a.P] : 0.f;
        }
    }
    // Requests that share a state are one sequence: the block of the first takes them all, in order, the others leave.
    bool shared = false;
    if (a.slots) {
        bool other = false, before = false;
        for (int j = tid; j < a.batch; j += kStepThreads)
            if (j != i && a.slots[j] == slot) {
                other = true;
                before |= j < i;
            }
        shared = __syncthreads_or(other);
        if (shared && __syncthreads_or(before)) return;
    }
    for (int j = i;;) {
        const float decay = expf(ld_any(a.g.ptr, a.g_dtype, j * a.g.sb + h * a.g.sh));
        float v[VEC], acc[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            v[e] = c + e < a.P ? ld<T>(a.v.ptr, j * a.v.sb + h * a.v.sh + c + e) : 0.f;
            acc[e] = 0.f;
        }
        const long long kq = j * a.k.sb + hq * a.k.sh, qq = j * a.q.sb + hq * a.q.sh;
#pragma unroll
        for (int r = 0; r < PASSES; ++r) {
            const int n = n0 + r * kRows;
            const bool in = n < a.N;
            const float k = in ? ld<T>(a.k.ptr, kq + n) : 0.f, q = in ? ld<T>(a.q.ptr, qq + n) : 0.f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                s[r][e] = fmaf(s[r][e], decay, __fmul_rn(k, v[e]));   // written out: the same bits in every variant
                acc[e] = fmaf(q, s[r][e], acc[e]);
            }
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
#pragma unroll
            for (int o = kLanes; o < 32; o <<= 1) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], o);
            if (lane < kLanes) part[warp][lane * VEC + e] = acc[e];
        }
        __syncthreads();
        if (tid < kStepColumns && oc < a.P) {
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < kStepThreads / 32; ++w) sum += part[w][tid];
            st<T>(a.o.ptr, j * a.o.sb + h * a.o.sh + oc, a.scale * sum);
        }
        if (!shared) break;
        bool more = false;                                       // the next request of this state
        for (int j0 = j + 1; j0 < a.batch && !more; j0 += kStepThreads) {
            const int cand = j0 + tid;
            const unsigned hit = __ballot_sync(0xffffffffu, cand < a.batch && a.slots[cand] == slot);
            __shared__ int first[kStepThreads / 32];
            if (lane == 0) first[warp] = hit ? j0 + warp * 32 + __ffs(hit) - 1 : a.batch;
            __syncthreads();
            int next = a.batch;
            for (int w = 0; w < kStepThreads / 32; ++w) next = min(next, first[w]);
            if (next < a.batch) {
                j = next;
                more = true;
            }
            __syncthreads();
        }
        if (!more) break;
    }
#pragma unroll
    for (int r = 0; r < PASSES; ++r) {
        const int n = n0 + r * kRows;
        if (n >= a.N || c >= a.P) continue;
        if constexpr (VEC == 4) __stcs(reinterpret_cast<float4 *>(base + (long long)n * a.P), make_float4(s[r][0], s[r][1], s[r][2], s[r][3]));
        else base[(long long)n * a.P] = s[r][0];
    }
}

}  // namespace uni
}  // namespace bissd
