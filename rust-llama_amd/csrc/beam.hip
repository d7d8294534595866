// beam.hip - beam search's choice on gfx950.
//
// A candidate of a group is a beam b and a token t with
//   rank = score_b + z_bt - log sum_u exp z_bu
// in f64 from the f32 logits (the exponentials f32, their sum f64); the best
// candidates in order, the lowest (b, t) of equal ones.  Within a beam the order is
// that of the logits, so a beam's logits are read once: for its sum and for its best tokens,
// which meet those of the other beams as f64 ranks.
#include "rlq_device.hpp"
#include "rlq_internal.hpp"

namespace rlq {

// Floats as whole numbers of the same order (-0 as 0).
constexpr uint32_t kLeast = 0x00800000u;  // of the floats above -infinity
__device__ __forceinline__ uint32_t beam_key(float z) {
    const uint32_t b = __float_as_uint(z == 0.0f ? 0.0f : z);
    return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float beam_value(uint32_t key) {
    return __uint_as_float((key >> 31) ? key ^ 0x80000000u : ~key);
}
// A token with its logit: the larger logit, then the lower token, first; never 0.
__device__ __forceinline__ uint64_t beam_pair(uint32_t key, uint32_t token) { return (uint64_t)key << 32 | (uint32_t)~token; }
__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
    const uint32_t hi = wave_max_u32((uint32_t)(v >> 32));
    return (uint64_t)hi << 32 | wave_max_u32((uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
}

// What workgroups hand each other is put there by exchanges (performed at the device's
// coherent level when they return) and read at that level.
__device__ __forceinline__ void beam_put(unsigned long long* to, unsigned long long v) {
    const unsigned long long old = __hip_atomic_exchange(to, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("" ::"v"(old) : "memory");
}
__device__ __forceinline__ unsigned long long beam_get(const unsigned long long* from) {
    return __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Whether this workgroup is the last of n; the count is left at 0.  What it has put is there.
__device__ __forceinline__ bool beam_last(uint32_t* count, uint32_t n, uint32_t* flag) {
    __syncthreads();
    if (threadIdx.x == 0) {
        const uint32_t old = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *flag = old == n - 1;
        if (*flag) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return *flag != 0;
}

// exp(x) for x <= 0, within 2^-22: x log2(e) in two f32, the lower one applied to the power.
__device__ __forceinline__ float beam_exp(float x) {
    const float hi = 1.44269502f, lo = 1.92596299e-8f;  // log2(e) in two f32
    x = fmaxf(x, -200.0f);  // (of -infinity the remainder is no number; both give 0)
    const float t = x * hi, r = __builtin_fmaf(x, lo, __builtin_fmaf(x, hi, -t));
    const float p = __builtin_amdgcn_exp2f(t);
    return __builtin_fmaf(p, r * 0.693147181f, p);
}

constexpr uint32_t kWaveMost = 256;  // candidates that a wave puts down at once
constexpr uint32_t kListMost = kSelectMaxBest + 4 * kWaveMost;

// A workgroup per chunk of a beam's row, 4 U logits a thread at a time in registers.
//   Sum: every wave about its own maximum.
//   Best: of the maxima of a lane's quarters (256 in a wave) the best'th largest is no larger than
//   the best'th largest logit of the wave; it is found bit by bit with ballots, and only the logits from it on,
//   a few more than `best`, are put into a list in LDS, where each counts those before it.
//   (Where very many are equal, they are taken one by one instead.)
// The last chunk of a row merges the chunks' sorted lists, a lane for each; the last row of a group
// the beams'.  One launch.
template <int U>
__global__ __launch_bounds__(256) void beam_select_kernel(SelectArgs a) {
    extern __shared__ __align__(16) unsigned long long buf[];
    __shared__ float wave_m[4];
    __shared__ double wave_sum[4];
    __shared__ uint32_t listed, flag;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = a.vocabulary, k = a.best;
    const uint32_t row = blockIdx.y, chunk = blockIdx.x, chunks = gridDim.x, group = row / a.beams;
    const float* z = a.logits + (uint64_t)row * a.stride;
    const float score = a.scores[row];
    const uint32_t t0 = chunk * a.chunk, t1 = V - t0 < a.chunk ? V : t0 + a.chunk;
    float m = -INFINITY;
    double sum = 0.0;
    bool bad = !(score < INFINITY);
    uint32_t have = 0;
    if (score > -INFINITY && !bad) {
        for (uint32_t s = t0; s < t1; s += 1024 * U) {
            float v[U][4];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t t = s + 4 * (tid + 256 * u);
                if (t + 3 < t1) {
                    const f32x4 f = *(const f32x4a4*)(z + t);
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[u][j] = f[j];
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[u][j] = t + j < t1 ? z[t + j] : -INFINITY;
                }
            }
            uint32_t key[U][4], quarter[4] = {0, 0, 0, 0};
            float top = -INFINITY;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    bad |= !(v[u][j] < INFINITY);
                    key[u][j] = beam_key(v[u][j]);
                    quarter[j] = key[u][j] > quarter[j] ? key[u][j] : quarter[j];
                    top = fmaxf(top, v[u][j]);
                }
            top = wave_max_dpp(top);
            if (top > -INFINITY) {  // (uniform)
                if (top > m) {
                    sum *= (double)beam_exp(m - top);
                    m = top;
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
                    sum += (double)((beam_exp(v[u][0] - m) + beam_exp(v[u][1] - m)) + (beam_exp(v[u][2] - m) + beam_exp(v[u][3] - m)));
            }
            // the list so far is in buf[0 .. have), sorted; a full one bounds what can follow
            uint32_t least = have == k ? (uint32_t)(buf[k - 1] >> 32) : kLeast;
            if (tid == 0) listed = have;
            __syncthreads();
            {
                // the largest t with `best` quarters or more of t at least
                uint32_t t = 0;
                for (int bit = 31; bit >= 0; --bit) {
                    const uint32_t c = t | 1u << bit;
                    uint32_t n = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) n += (uint32_t)__builtin_popcountll(__ballot(quarter[j] >= c));
                    if (n >= k) t = c;
                }
                least = t > least ? t : least;
            }
            uint32_t n = 0;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) n += (uint32_t)__builtin_popcountll(__ballot(key[u][j] >= least));
            if (n <= kWaveMost) {
                uint32_t at = 0;
                if (lane == 0 && n) at = atomicAdd(&listed, n);
                at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const bool take = key[u][j] >= least;
                        const unsigned long long mask = __ballot(take);
                        if (!mask) continue;
                        if (take) buf[at + __builtin_popcountll(mask & ((1ull << lane) - 1))] = beam_pair(key[u][j], s + 4 * (tid + 256 * u) + j);
                        at += (uint32_t)__builtin_popcountll(mask);
                    }
            } else {
                uint64_t before = ~0ull;
                for (uint32_t i = 0; i < k; ++i) {
                    uint64_t best = 0;
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint64_t p = beam_pair(key[u][j], s + 4 * (tid + 256 * u) + j);
                            if (key[u][j] >= least && p < before && p > best) best = p;
                        }
                    best = wave_max_u64(best);
                    if (!best) break;
                    if (lane == 0) buf[atomicAdd(&listed, 1u)] = best;
                    before = best;
                }
            }
            __syncthreads();
            // each of the list counts those before it (all are different)
            const uint32_t all = listed;
            constexpr int kMine = (kListMost + 255) / 256;
            uint64_t mine[kMine];
            uint32_t place[kMine];
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const uint32_t c = tid + 256 * i;
                mine[i] = c < all ? buf[c] : 0;
                place[i] = 0;
                if (256u * i >= all) continue;  // (uniform)
                for (uint32_t j = 0; j < all; ++j) place[i] += buf[j] > mine[i];
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kMine; ++i)
                if (mine[i] && place[i] < k) buf[place[i]] = mine[i];
            have = all < k ? all : k;
            __syncthreads();
        }
    }
    bad = __syncthreads_or(bad);
    sum = wave_sum_f64(sum);
    if (lane == 0) wave_m[wave] = m, wave_sum[wave] = sum;
    __syncthreads();
    m = fmaxf(fmaxf(wave_m[0], wave_m[1]), fmaxf(wave_m[2], wave_m[3]));
    sum = 0.0;
    for (int w = 0; w < 4; ++w)
        if (wave_m[w] > -INFINITY) sum += wave_sum[w] * (double)beam_exp(wave_m[w] - m);
    if (bad) sum = NAN;

    // the row: every chunk's list
    if (chunks > 1) {
        unsigned long long* put = a.lists + ((uint64_t)row * chunks + chunk) * (k + 2);
        if (tid < k) beam_put(put + tid, tid < have ? buf[tid] : 0);
        if (tid == k) beam_put(put + k, __float_as_uint(m));
        if (tid == k + 1) beam_put(put + k + 1, (unsigned long long)__double_as_longlong(sum));
        if (!beam_last(a.count + row, chunks, &flag)) return;
        const unsigned long long* lists = a.lists + (uint64_t)row * chunks * (k + 2);
        for (uint32_t i = tid; i < chunks * (k + 2); i += 256) {
            const uint32_t c = i / (k + 2), j = i - c * (k + 2);
            const unsigned long long x = beam_get(lists + i);
            if (j < k) buf[c * k + j] = x;
            else buf[chunks * k + 2 * c + (j - k)] = x;
        }
        __syncthreads();
    }
    double rank = -INFINITY;  // of place `lane` in the row
    int32_t token = -1;
    if (wave == 0) {
        uint64_t pair = lane < have ? buf[lane] : 0;
        if (chunks > 1) {
            const bool some = lane < chunks;
            const float cm = some ? __uint_as_float((uint32_t)buf[chunks * k + 2 * lane]) : -INFINITY;
            const double cs = some ? __longlong_as_double((long long)buf[chunks * k + 2 * lane + 1]) : 0.0;
            m = wave_max_dpp(cm);
            // (a sum that is no number stays one)
            sum = wave_sum_f64(cs != cs ? cs : cm > -INFINITY ? cs * (double)beam_exp(cm - m) : 0.0);
            uint32_t next = 1;
            uint64_t head = some ? buf[lane * k] : 0;
            pair = 0;
            for (uint32_t i = 0; i < k; ++i) {
                const uint64_t best = wave_max_u64(head);
                if (!best) break;
                if (lane == i) pair = best;
                if (head == best) head = next < k ? buf[lane * k + next] : 0, ++next;
            }
        }
        if (sum != sum) rank = NAN;
        else if (pair) rank = (double)score - ((double)m + log(sum)) + (double)beam_value((uint32_t)(pair >> 32)), token = (int32_t)~(uint32_t)pair;
    }

    // the group: every beam's
    int32_t parent = token < 0 ? -1 : 0;
    if (a.beams > 1) {
        unsigned long long* put = a.ranks + (uint64_t)row * 2 * k;
        if (wave == 0 && lane < k) {
            beam_put(put + lane, (unsigned long long)__double_as_longlong(rank));
            beam_put(put + k + lane, (uint32_t)token);
        }
        if (!beam_last(a.count + (uint64_t)a.groups * a.beams + group, a.beams, &flag)) return;
        const unsigned long long* ranks = a.ranks + (uint64_t)group * a.beams * 2 * k;
        uint32_t* tokens = (uint32_t*)(buf + a.beams * k);
        for (uint32_t i = tid; i < a.beams * 2 * k; i += 256) {
            const uint32_t b = i / (2 * k), j = i - b * 2 * k;
            const unsigned long long x = beam_get(ranks + i);
            if (j < k) buf[b * k + j] = x;
            else tokens[b * k + j - k] = (uint32_t)x;
        }
        __syncthreads();
        if (wave != 0) return;
        const unsigned long long* list = buf + lane * k;
        const bool some = lane < a.beams;
        double head = some ? __longlong_as_double((long long)list[0]) : -INFINITY;
        const bool off = __ballot(head != head) != 0;
        uint32_t next = 1;
        rank = off ? NAN : -INFINITY, token = parent = -1;
        for (uint32_t i = 0; i < k && !off; ++i) {
            const double best = wave_max_f64(head);
            if (!(best > -INFINITY)) break;
            const int b = __builtin_ctzll(__ballot(head == best));  // the lowest beam of equal ones
            if (lane == i) rank = best, parent = b, token = (int32_t)tokens[b * k + __builtin_amdgcn_readlane((int)next, b) - 1];
            if ((int)lane == b) head = next < k ? __longlong_as_double((long long)list[next]) : -INFINITY, ++next;
        }
    } else if (wave != 0) {
        return;
    }
    if (__ballot(rank != rank)) {
        rank = -INFINITY, token = parent = -1;
        if (lane == 0) report_error(a.err_word, model_key(a.group0 + group, kStOOut, 0));
    }
    if (lane < k) {
        const uint64_t o = (uint64_t)group * k + lane;
        a.out_scores[o] = (float)rank, a.parents[o] = parent, a.tokens[o] = token;
    }
}

// Logits of a thread at a time, and of a workgroup: few rows are cut finer, to fill the CUs (4 rows of 128256
// tokens: 252 workgroups); at most 64 chunks, which a wave's lanes merge.
static uint32_t select_unroll(uint64_t rows, uint64_t vocabulary) {
    const uint64_t chunks = (vocabulary + 2047) / 2048;
    return rows * chunks <= 1024 && chunks <= 64 ? 2 : rows * chunks <= 2048 && chunks <= 128 ? 4 : 8;
}
static uint32_t select_chunk(uint64_t rows, uint64_t vocabulary) {
    const uint64_t unit = 1024 * select_unroll(rows, vocabulary);
    uint64_t n = (vocabulary + unit - 1) / unit;
    n = n < 64 ? n : 64;
    return (uint32_t)(((vocabulary + n - 1) / n + 3) / 4 * 4);
}
static uint64_t select_chunks(uint64_t rows, uint64_t vocabulary) {
    const uint64_t c = select_chunk(rows, vocabulary);
    return (vocabulary + c - 1) / c;
}
size_t beam_select_bytes(uint64_t rows, uint64_t vocabulary, uint64_t best) {
    return rows * (select_chunks(rows, vocabulary) * (best + 2) + 2 * best) * sizeof(unsigned long long);
}

hipError_t launch_beam_select(SelectArgs a, void* scratch, hipStream_t s) {
    if (a.groups == 0 || a.groups > 65535 || a.beams == 0 || a.beams > kSelectMaxBeams || a.best == 0 ||
        a.best > kSelectMaxBest || a.vocabulary == 0)
        return hipErrorInvalidValue;
    const uint64_t rows = (uint64_t)a.groups * a.beams, chunks = select_chunks(rows, a.vocabulary);
    a.chunk = select_chunk(rows, a.vocabulary);
    a.ranks = (unsigned long long*)scratch;
    a.lists = a.ranks + rows * 2 * a.best;
    uint64_t words = chunks > 1 ? chunks * (a.best + 2) : 0;
    if (words < kListMost) words = kListMost;
    const uint64_t of_beams = ((uint64_t)a.beams * a.best * 3 + 1) / 2;  // (at most 48 KB)
    if (words < of_beams) words = of_beams;
    for (uint64_t g = 0; g < a.groups;) {  // (a grid's second dimension has 65535 workgroups)
        const uint64_t n = a.groups - g < 65535 / a.beams ? a.groups - g : 65535 / a.beams;
        SelectArgs p = a;
        p.logits += g * a.beams * a.stride, p.scores += g * a.beams;
        p.out_scores += g * a.best, p.parents += g * a.best, p.tokens += g * a.best;
        p.group0 = (uint32_t)g, p.groups = (uint32_t)n;
        const dim3 grid((uint32_t)chunks, (uint32_t)(n * a.beams)), block(256);
        const size_t lds = words * sizeof(unsigned long long);
        switch (select_unroll(rows, a.vocabulary)) {
            case 2: hipLaunchKernelGGL(beam_select_kernel<2>, grid, block, lds, s, p); break;
            case 4: hipLaunchKernelGGL(beam_select_kernel<4>, grid, block, lds, s, p); break;
            default: hipLaunchKernelGGL(beam_select_kernel<8>, grid, block, lds, s, p); break;
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        g += n;
    }
    return hipSuccess;
}

}  // namespace rlq
