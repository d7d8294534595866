// beam.hip - beam search's choice on gfx950.
//
// A candidate of a group is a beam b and a token t with
//   rank = score_b + z_bt - log sum_u exp z_bu
// in f64 from the f32 logits (the exponentials f32, their sum f64); the best
// candidates in order, the lowest (b, t) of equal ones.  Within a beam the order is
// that of the logits.
#include "rlq_device.hpp"
#include "rlq_internal.hpp"

namespace rlq {

// Floats as whole numbers of the same order (-0 as 0; 0: less than any).
__device__ __forceinline__ uint32_t beam_key(float z) {
    const uint32_t b = __float_as_uint(z == 0.0f ? 0.0f : z);
    return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float beam_value(uint32_t key) {
    return __uint_as_float((key >> 31) ? key ^ 0x80000000u : ~key);
}
__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
    for (int m = 1; m < 64; m <<= 1) {
        const uint64_t o = __shfl_xor(v, m, 64);
        v = o > v ? o : v;
    }
    return v;
}

// A beam's best tokens, one workgroup per beam: the log of the sum, then one pass
// over the row for each place.
__global__ __launch_bounds__(1024) void beam_row_kernel(SelectArgs a) {
    __shared__ uint64_t most[16];
    __shared__ double sums[16];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint64_t row = blockIdx.x;
    const float* z = a.logits + row * a.stride;
    double* rank = a.rank + row * a.best;
    int32_t* token = a.token + row * a.best;
    const float score = a.scores[row];
    uint64_t top = 0;
    int bad = !(score < INFINITY);
    if (score > -INFINITY) {
        for (uint32_t i = tid; i < a.vocabulary; i += 1024) {
            const float v = z[i];
            bad |= !(v < INFINITY);
            const uint64_t key = (uint64_t)beam_key(v) << 32 | (uint32_t)~i;
            if (v > -INFINITY) top = key > top ? key : top;
        }
    }
    bad = __syncthreads_or(bad);
    auto block_max = [&](uint64_t v) {
        v = wave_max_u64(v);
        __syncthreads();
        if (lane == 0) most[wave] = v;
        __syncthreads();
        for (int w = 0; w < 16; ++w) v = most[w] > v ? most[w] : v;
        return v;
    };
    top = block_max(top);
    if (bad && tid == 0) report_error(a.err_word, model_key((uint32_t)(row / a.beams), kStOOut, 0));
    if (bad || top == 0) {
        for (uint32_t i = tid; i < a.best; i += 1024) rank[i] = bad ? NAN : -INFINITY, token[i] = -1;
        return;
    }
    const float m = beam_value((uint32_t)(top >> 32));
    double sum = 0.0;
    for (uint32_t i = tid; i < a.vocabulary; i += 1024) sum += (double)expf(z[i] - m);
    sum = wave_sum_f64(sum);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    sum = 0.0;
    for (int w = 0; w < 16; ++w) sum += sums[w];
    const double offset = (double)score - ((double)m + log(sum));
    for (uint32_t i = 0; i < a.best; ++i) {
        if (tid == 0) {
            rank[i] = top ? offset + (double)beam_value((uint32_t)(top >> 32)) : -INFINITY;
            token[i] = top ? (int32_t)~(uint32_t)top : -1;
        }
        uint64_t next = 0;
        if (top)
            for (uint32_t j = tid; j < a.vocabulary; j += 1024) {
                const uint64_t key = (uint64_t)beam_key(z[j]) << 32 | (uint32_t)~j;
                if (z[j] > -INFINITY && key < top) next = key > next ? key : next;
            }
        top = block_max(next);
    }
}

// A group's best candidates of those of its beams.
__global__ __launch_bounds__(256) void beam_group_kernel(SelectArgs a) {
    __shared__ double best_of[4];
    __shared__ uint32_t where_of[4];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.beams * a.best;
    const uint64_t group = blockIdx.x;
    const double* rank = a.rank + group * n;
    const int32_t* token = a.token + group * n;
    int bad = 0;
    for (uint32_t i = tid; i < n; i += 256) bad |= rank[i] != rank[i];
    bad = __syncthreads_or(bad);
    double last = INFINITY;
    uint32_t at = 0;
    for (uint32_t k = 0; k < a.best; ++k) {
        double top = -INFINITY;
        uint32_t where = 0xffffffffu;
        if (!bad)
            for (uint32_t i = tid; i < n; i += 256) {
                const double r = rank[i];
                const bool left = r > -INFINITY && (k == 0 || r < last || (r == last && i > at));
                if (left && r > top) top = r, where = i;
            }
        for (int m = 1; m < 64; m <<= 1) {
            const double o = __shfl_xor(top, m, 64);
            const uint32_t w = (uint32_t)__shfl_xor((int)where, m, 64);
            if (o > top || (o == top && w < where)) top = o, where = w;
        }
        __syncthreads();
        if (lane == 0) best_of[wave] = top, where_of[wave] = where;
        __syncthreads();
        for (int w = 0; w < 4; ++w)
            if (best_of[w] > top || (best_of[w] == top && where_of[w] < where)) top = best_of[w], where = where_of[w];
        if (tid == 0) {
            const uint64_t o = group * a.best + k;
            const bool some = where != 0xffffffffu;
            a.out_scores[o] = some ? (float)top : -INFINITY;
            a.parents[o] = some ? (int32_t)(where / a.best) : -1;
            a.tokens[o] = some ? token[where] : -1;
        }
        last = top, at = where;
    }
}

size_t beam_select_bytes(uint64_t rows, uint64_t best) { return rows * best * (sizeof(double) + sizeof(int32_t)); }

hipError_t launch_beam_select(SelectArgs a, void* scratch, hipStream_t s) {
    if (a.groups == 0 || a.groups > 65535 || a.beams == 0 || a.beams > kSelectMaxBeams || a.best == 0 ||
        a.best > kSelectMaxBest || a.vocabulary == 0)
        return hipErrorInvalidValue;
    const uint64_t rows = (uint64_t)a.groups * a.beams;
    a.rank = (double*)scratch;
    a.token = (int32_t*)(a.rank + rows * a.best);
    hipLaunchKernelGGL(beam_row_kernel, dim3((uint32_t)rows), dim3(1024), 0, s, a);
    hipLaunchKernelGGL(beam_group_kernel, dim3(a.groups), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace rlq
