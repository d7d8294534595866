// beam.hip - beam search's choice on gfx950.
//
// A candidate of a group is a beam b and a token t with
//   rank = score_b + z_bt - log sum_u exp z_bu
// in f64 from the f32 logits (the exponentials f32, their sum f64); the best
// candidates in order.  Within a beam the order is that of the logits (the lower token of equal ones), of equal ranks
// the lower beam's is first.  So a beam's logits are read once: for its sum and for its best tokens,
// which meet those of the other beams as f64 ranks.
#include "rlq_device.hpp"
#include "rlq_internal.hpp"

namespace rlq {

// Floats as whole numbers of the same order (-0 as 0).
constexpr uint32_t kLeast = 0x00800000u;  // of the floats above -infinity
__device__ __forceinline__ uint32_t beam_key(float z) {
    const uint32_t b = __float_as_uint(z + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
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

constexpr uint32_t kFound = 512;       // candidates of a group that are ranked by counting
constexpr uint32_t kWaveMost = 256;  // candidates that a wave puts down at once
constexpr uint32_t kListMost = kSelectMaxBest + kWaveMost;  // of a wave's list

// LDS that a wave writes and reads by itself: its operations are performed in order.
__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The first k of n different numbers in LDS, in descending order at its beginning; by the
// lanes `lane` of `lanes` (a wave, or all waves of the workgroup with `join` between), up to M numbers a lane.  Each
// number counts those before it.
template <int M, class Join>
__device__ __forceinline__ void keep_best(unsigned long long* list, uint32_t n, uint32_t k, uint32_t lane, uint32_t lanes,
                                          Join&& join) {
    uint64_t mine[M];
    uint32_t place[M];
#pragma unroll
    for (int i = 0; i < M; ++i) {
        mine[i] = lane + lanes * i < n ? list[lane + lanes * i] : 0;
        place[i] = 0;
    }
#pragma unroll
    for (int i = 0; i < M; ++i) {
        if (lanes * i >= n) continue;  // (uniform)
        uint32_t j = 0;
        for (; j + 8 <= n; j += 8) {
            uint64_t o[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) o[u] = list[j + u];
#pragma unroll
            for (int u = 0; u < 8; ++u) place[i] += o[u] > mine[i];
        }
        for (; j < n; ++j) place[i] += list[j] > mine[i];
    }
    join();
#pragma unroll
    for (int i = 0; i < M; ++i)
        if (mine[i] && place[i] < k) list[place[i]] = mine[i];
    join();
}

// A number that k of the wave's 64 N keys reach, and no more than k + 3 where their bits allow it; 0 if there are no k
// above 0.  Bit by bit with ballots.
template <int N>
__device__ __forceinline__ uint32_t bound_of(const uint32_t (&key)[N], uint32_t k) {
    uint32_t t = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t c = t | 1u << bit;
        uint32_t n = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) n += (uint32_t)__builtin_popcountll(__ballot(key[j] >= c));
        if (n >= k) t = c;
        if (n >= k && n < k + 4) break;
    }
    return t;
}

// f64 ranks as whole numbers of the same order; 0: none (-infinity).  kNoRank: a rank that is no number.
constexpr uint64_t kNoRank = ~0ull;
__device__ __forceinline__ uint64_t rank_key(double r) {
    if (!(r > -INFINITY)) return r != r ? kNoRank : 0;
    const uint64_t b = (uint64_t)__double_as_longlong(r + 0.0);
    return b ^ ((uint64_t)((int64_t)b >> 63) | 1ull << 63);
}
__device__ __forceinline__ double rank_value(uint64_t key) {
    return __longlong_as_double((long long)((key >> 63) ? key ^ 1ull << 63 : ~key));
}

// Lists of k numbers in descending order, one of each lane with `some` (0: no more), merged by a wave: lane i gets the
// i'th largest (0: none), the lane that it is of, the lowest of equal ones, and its place there.  A round
// looks for the largest upper half; only where several lanes have it the lower halves decide.
__device__ __forceinline__ void merge_lists(const unsigned long long* list, bool some, uint32_t k, uint64_t& key, uint32_t& from,
                                            uint32_t& place) {
    const uint32_t lane = threadIdx.x & 63;
    uint64_t head = some ? list[0] : 0, after = some && k > 1 ? list[1] : 0;
    uint32_t at = 0;
    key = 0, from = place = 0;
    for (uint32_t i = 0; i < k; ++i) {
        const uint32_t hi = (uint32_t)(head >> 32), best = wave_max_u32(hi);
        if (best == 0) break;
        unsigned long long mask = __ballot(hi == best);
        if (mask & (mask - 1)) {
            const uint32_t lo = hi == best ? (uint32_t)head : 0, low = wave_max_u32(lo);
            mask = __ballot(hi == best && lo == low);
        }
        const int b = __builtin_ctzll(mask);
        const uint64_t k0 = (uint64_t)best << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)head, b);
        const uint32_t p = (uint32_t)__builtin_amdgcn_readlane((int)at, b);
        if (lane == i) key = k0, from = (uint32_t)b, place = p;
        if ((int)lane == b) {
            head = after, ++at;
            after = at + 1 < k ? list[at + 1] : 0;
        }
    }
}

// A workgroup per chunk of a beam's row; its waves go through it 256 U logits at a time, the next on their
// way, each by itself:
//   Sum: about the wave's own maximum.
//   Best: of the maxima of a lane's quarters (256 in a wave) the k'th largest is no larger than the
//   k'th largest logit; it is searched bit by bit with ballots, until k to k + 3 of them reach it.  Only logits from
//   it on, and from the k'th best so far, go to the wave's list in LDS (a few more than k at first, then fewer and
//   fewer).  Where very many are equal, they are taken one by one instead.
// The waves' lists are joined and put where every workgroup can read them.  Where a group's lists are few (256, 32 KB)
// its last workgroup takes all of them into LDS: of their first ranks the best'th bounds what can be chosen, and
// what reaches it, some tens of candidates, is ranked by counting.  Else the last chunk of a row merges the row's
// sorted lists, a lane for each, and the last row of the group the beams'.  One launch.
//
// Bound: four beams of 128256 tokens, the best 8: 14.9 us, of which the loads are 2.3, sums and lists 2.2, the waves'
// lists 1.6, putting and counting 3.4 (252 workgroups count at one place), the choice 5.  16 groups of
// eight beams of 151936 tokens, the best 16: 38 us; the loads alone 13.4 (5.8 TB/s), sums and lists 11 beside them
// (30 VALU instructions a logit, eight of them the exponential; 23 of them, or twice the waves, take as long), then
// 14 of joining.
template <int U>
__global__ __launch_bounds__(256) void beam_select_kernel(SelectArgs a) {
    extern __shared__ __align__(16) unsigned long long buf[];
    __shared__ float wave_m[4];
    __shared__ double wave_sum[4];
    __shared__ uint32_t wave_have[4], flag;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = a.vocabulary, k = a.best;
    const uint32_t row = blockIdx.y, chunk = blockIdx.x, chunks = gridDim.x, group = row / a.beams;
    const float* z = a.logits + (uint64_t)row * a.stride;
    const float score = a.scores[row];
    const uint32_t t0 = chunk * a.chunk, t1 = V - t0 < a.chunk ? V : t0 + a.chunk;
    float m = -INFINITY;
    double sum = 0.0;
    int bad = !(score < INFINITY);
    uint32_t have = 0, least = kLeast;
    if (score > -INFINITY && !bad) {
        unsigned long long* list = buf + wave * kListMost;
        const uint32_t mine = 4 * tid;  // of every 1024: a wave's are together
        f32x4 v[U];
        auto load = [&](uint32_t s) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t t = s + 1024 * u + mine;
                if (t + 3 < t1) {
                    v[u] = __builtin_nontemporal_load((const f32x4a4*)(z + t));
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[u][j] = t + j < t1 ? z[t + j] : -INFINITY;
                }
            }
        };
        load(t0);
        for (uint32_t s = t0; s < t1; s += 1024 * U) {
            uint32_t key[U][4], quarter[4] = {0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < U; ++u) {
                bad |= __builtin_isunordered(v[u][0], v[u][1]) || __builtin_isunordered(v[u][2], v[u][3]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    key[u][j] = beam_key(v[u][j]);
                    quarter[j] = key[u][j] > quarter[j] ? key[u][j] : quarter[j];
                }
            }
            const uint32_t a01 = quarter[0] > quarter[1] ? quarter[0] : quarter[1];
            const uint32_t a23 = quarter[2] > quarter[3] ? quarter[2] : quarter[3];
            const uint32_t highest = wave_max_u32(a01 > a23 ? a01 : a23);
            const bool some = highest >= kLeast;  // (uniform in the wave)
            if (some) {
                const float top = beam_value(highest);
                bad |= !(top < INFINITY);
                if (top > m) {
                    sum *= (double)beam_exp(m - top);
                    m = top;
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
                    sum += (double)((beam_exp(v[u][0] - m) + beam_exp(v[u][1] - m)) + (beam_exp(v[u][2] - m) + beam_exp(v[u][3] - m)));
            }
            if (t1 - s > 1024 * U) load(s + 1024 * U);
            if (highest < least || !some) continue;
            // the k'th best so far bounds what can follow; before there is one, or where it lets too much through, the
            // k'th largest quarter does
            uint32_t at = have;
            auto put = [&] {
                at = have;
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const bool take = key[u][j] >= least;
                        const unsigned long long mask = __ballot(take);
                        if (!mask) continue;
                        const uint32_t to = at + (uint32_t)__builtin_popcountll(mask & ((1ull << lane) - 1));
                        if (take && to < kListMost) list[to] = beam_pair(key[u][j], s + 1024 * u + mine + j);
                        at += (uint32_t)__builtin_popcountll(mask);
                    }
            };
            if (least > kLeast) put();
            if (least == kLeast || at > kListMost) {
                const uint32_t t = bound_of<4>(quarter, k);
                least = t > least ? t : least;
                put();
            }
            if (at > kListMost) {  // very many equal ones
                at = have;
                uint64_t before = ~0ull;
                for (uint32_t i = 0; i < k; ++i) {
                    uint64_t best = 0;
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint64_t p = beam_pair(key[u][j], s + 1024 * u + mine + j);
                            if (key[u][j] >= least && p < before && p > best) best = p;
                        }
                    best = wave_max_u64(best);
                    if (!best) break;
                    if (lane == 0) list[at] = best;
                    ++at, before = best;
                }
            }
            wave_order();
            // sorted when there are k for the first time, and before another wave's worth would not fit
            if ((have < k && at >= k) || at > kSelectMaxBest) {
                keep_best<(int)(kListMost + 63) / 64>(list, at, k, lane, 64, [] { wave_order(); });
                at = at < k ? at : k;
                if (at == k) least = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(list[k - 1] >> 32));
            }
            have = at;
        }
        if (have > k) {
            keep_best<1>(list, have, k, lane, 64, [] { wave_order(); });
            have = k;
        }
    }
    sum = wave_sum_f64(sum);
    if (lane == 0) wave_m[wave] = m, wave_sum[wave] = sum, wave_have[wave] = have;
    bad = __syncthreads_or(bad);
    m = fmaxf(fmaxf(wave_m[0], wave_m[1]), fmaxf(wave_m[2], wave_m[3]));
    sum = 0.0;
    for (int w = 0; w < 4; ++w)
        if (wave_m[w] > -INFINITY) sum += wave_sum[w] * (double)beam_exp(wave_m[w] - m);
    if (bad) sum = NAN;
    {  // the waves' lists, one behind the other
        uint32_t at = 0;
        for (uint32_t w = 0; w < wave; ++w) at += wave_have[w];
        const unsigned long long pair = lane < have ? buf[wave * kListMost + lane] : 0;
        const uint32_t all = wave_have[0] + wave_have[1] + wave_have[2] + wave_have[3];
        __syncthreads();
        if (lane < have) buf[at + lane] = pair;
        __syncthreads();
        keep_best<1>(buf, all, k, tid, 256, [] { __syncthreads(); });
        have = all < k ? all : k;
    }

    // the row: every chunk's list.  Few beams: of all of the group at once
    const bool once = a.once;
    if (chunks > 1 || once) {
        const uint32_t words = chunks * (k + 2), mine = (row - group * a.beams) * words + chunk * (k + 2);
        unsigned long long* put = a.lists + (uint64_t)group * a.beams * words + mine;
        if (tid < k) beam_put(put + tid, tid < have ? buf[tid] : 0);
        if (tid == k) beam_put(put + k, __float_as_uint(m));
        if (tid == k + 1) beam_put(put + k + 1, (unsigned long long)__double_as_longlong(sum));
        if (!beam_last(once ? a.count + group : a.count + row, once ? chunks * a.beams : chunks, &flag)) return;
        const unsigned long long* lists = put - (once ? mine : chunk * (k + 2));
        const uint32_t n = (once ? a.beams : 1) * words;
        for (uint32_t i = tid; i < n; i += 8 * 256) {
            unsigned long long x[8];
#pragma unroll
            for (uint32_t u = 0; u < 8; ++u) x[u] = i + 256 * u < n ? beam_get(lists + i + 256 * u) : 0;
#pragma unroll
            for (uint32_t u = 0; u < 8; ++u)
                if (i + 256 * u < n) buf[i + 256 * u] = x[u];
        }
        __syncthreads();
    }
    // score less the log of the sum, of a row whose chunks' lists are at `lists` (no number: an error)
    auto row_offset = [&](const unsigned long long* lists, float of) {
        const bool some = lane < chunks;
        const unsigned long long* list = lists + lane * (k + 2);
        const float cm = some ? __uint_as_float((uint32_t)list[k]) : -INFINITY;
        const double cs = some ? __longlong_as_double((long long)list[k + 1]) : 0.0;
        const float top = wave_max_dpp(cm);
        // (a sum that is no number stays one; no logits at all: their ranks are not made)
        const double all = wave_sum_f64(cs != cs ? cs : cm > -INFINITY ? cs * (double)beam_exp(cm - top) : 0.0);
        return all != all ? (double)NAN : top > -INFINITY ? (double)of - ((double)top + log(all)) : 0.0;
    };
    auto rank_of = [](double offset, uint64_t pair) { return pair ? rank_key(offset + (double)beam_value((uint32_t)(pair >> 32))) : 0; };
    if (once) {
        // all lists of the group at once, a thread for each
        const uint32_t words = chunks * (k + 2), lists = a.beams * chunks;
        double* offset = (double*)(buf + a.beams * words);
        unsigned long long* heads = (unsigned long long*)(offset + kSelectMaxBeams);
        unsigned long long* found = heads + 256;
        uint32_t* found_at = (uint32_t*)(found + kFound);
        auto out = [&](uint32_t p, uint64_t r, uint32_t at) {
            const uint64_t to = (uint64_t)group * k + p;
            const uint32_t l = at / 64;
            a.out_scores[to] = r ? (float)rank_value(r) : -INFINITY;
            a.parents[to] = r ? (int32_t)(l / chunks) : -1;
            a.tokens[to] = r ? (int32_t)~(uint32_t)buf[l * (k + 2) + at % 64] : -1;
        };
        // of two places of equal rank, whether the first is (a score far from the logits rounds them away): the lower
        // beam's, then the larger logit's, then the lower token's
        auto first_of = [&](uint32_t x, uint32_t y) {
            const uint32_t bx = x / 64 / chunks, by = y / 64 / chunks;
            return bx != by ? bx < by : buf[x / 64 * (k + 2) + x % 64] > buf[y / 64 * (k + 2) + y % 64];
        };
        for (uint32_t b = wave; b < a.beams; b += 4) {
            const double o = row_offset(buf + b * words, a.scores[(uint64_t)group * a.beams + b]);
            if (lane == 0) offset[b] = o;
        }
        if (tid == 0) wave_have[0] = 0;
        __syncthreads();
        const double o = tid < lists ? offset[tid / chunks] : 0.0;
        heads[tid] = tid < lists ? rank_of(o, buf[tid * (k + 2)]) : 0;
        const bool off = __syncthreads_or(o != o);
        if (off) {
            if (tid == 0) report_error(a.err_word, model_key(a.group0 + group, kStOOut, 0));
            for (uint32_t p = tid; p < k; p += 256) out(p, 0, 0);
            return;
        }
        // of the heads, k to k + 3 reach `bound` (all waves find it)
        uint32_t top[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) top[u] = (uint32_t)(heads[lane + 64 * u] >> 32);
        const uint64_t bound = (uint64_t)bound_of<4>(top, k) << 32;
        const uint64_t least_rank = bound > 1 ? bound : 1;
        // their lists, the lanes a list's places: every fourth list a wave
        uint32_t turn = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            unsigned long long reach = __ballot(top[u] >= (uint32_t)(bound >> 32) && top[u] > 0);
            for (; reach; reach &= reach - 1, ++turn) {
                if (turn % 4 != wave) continue;
                const uint32_t l = 64 * u + (uint32_t)__builtin_ctzll(reach);
                const uint64_t r = lane < k ? rank_of(offset[l / chunks], buf[l * (k + 2) + lane]) : 0;
                const unsigned long long mask = __ballot(r >= least_rank);
                uint32_t at = 0;
                if (lane == 0) at = atomicAdd(&wave_have[0], (uint32_t)__builtin_popcountll(mask));
                at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at) + lane;  // (a list's first places reach it)
                if (r >= least_rank && at < kFound) found[at] = r, found_at[at] = l * 64 + lane;
            }
        }
        __syncthreads();
        const uint32_t n = wave_have[0];
        if (n <= kFound) {
            if (wave != 0) return;
            uint32_t left = n;
            if (n > 64) {  // those that reach the k'th of them
                constexpr int kMine = kFound / 64;
                uint64_t r[kMine];
                uint32_t hi[kMine], at[kMine];
#pragma unroll
                for (int u = 0; u < kMine; ++u) {
                    const uint32_t c = lane + 64 * u;
                    r[u] = c < n ? found[c] : 0, at[u] = c < n ? found_at[c] : 0;
                    hi[u] = (uint32_t)(r[u] >> 32);
                }
                const uint32_t t = bound_of<kMine>(hi, k);
                wave_order();
                left = 0;
#pragma unroll
                for (int u = 0; u < kMine; ++u) {
                    const bool take = hi[u] >= t && r[u];
                    const unsigned long long mask = __ballot(take);
                    const uint32_t to = left + (uint32_t)__builtin_popcountll(mask & ((1ull << lane) - 1));
                    if (take) found[to] = r[u], found_at[to] = at[u];
                    left += (uint32_t)__builtin_popcountll(mask);
                }
                wave_order();
            }
            for (uint32_t c = lane; c < left; c += 64) {
                const uint64_t mine = found[c];
                const uint32_t where = found_at[c];
                uint32_t p = 0, same = 0;
#pragma unroll 8
                for (uint32_t j = 0; j < left; ++j) p += found[j] > mine, same += found[j] == mine;
                if (same > 1)
                    for (uint32_t j = 0; j < left; ++j) p += found[j] == mine && first_of(found_at[j], where);
                if (p < k) out(p, mine, where);
            }
            for (uint32_t p = left + lane; p < k; p += 64) out(p, 0, 0);
            return;
        }
        // very many ranks between the best heads: a place at a time
        const unsigned long long* list = buf + tid * (k + 2);
        uint64_t head = heads[tid];
        uint32_t at = 0;
        __syncthreads();
        for (uint32_t i = 0; i < k; ++i) {
            const uint64_t best = wave_max_u64(head);
            if (lane == 0) heads[wave] = best;
            __syncthreads();
            uint64_t most = 0;
            for (int w = 0; w < 4; ++w) most = heads[w] > most ? heads[w] : most;
            // of equal ones the lowest beam's, and its largest logit (two tokens are never the same pair)
            const bool equal = head == most && most > 0;
            const unsigned long long mask = __ballot(equal);
            if (lane == 0) heads[4 + wave] = mask ? (wave * 64 + (uint32_t)__builtin_ctzll(mask)) / chunks : kSelectMaxBeams;
            __syncthreads();
            uint32_t beam = kSelectMaxBeams;
            for (int w = 3; w >= 0; --w) beam = heads[4 + w] < kSelectMaxBeams ? (uint32_t)heads[4 + w] : beam;
            const uint64_t pair = equal && tid / chunks == beam ? list[at] : 0, largest = wave_max_u64(pair);
            if (lane == 0) heads[8 + wave] = largest;
            __syncthreads();
            uint64_t first = 0;
            for (int w = 0; w < 4; ++w) first = heads[8 + w] > first ? heads[8 + w] : first;
            if (most == 0) {
                if (tid == 0) out(i, 0, 0);
            } else if (pair == first) {
                out(i, most, tid * 64 + at);
                ++at, head = at < k ? rank_of(o, list[at]) : 0;
            }
            __syncthreads();
        }
        return;
    }
    uint64_t rank = 0;
    int32_t token = -1;
    unsigned long long* ranks = buf;  // [beams][k], then the tokens
    uint32_t* tokens = (uint32_t*)(buf + a.beams * k);
    if (wave == 0) {
        uint64_t pair = lane < have ? buf[lane] : 0;
        double o = sum != sum ? (double)NAN : m > -INFINITY ? (double)score - ((double)m + log(sum)) : 0.0;
        if (chunks > 1) {
            uint32_t from, place;
            o = row_offset(buf, score);
            merge_lists(buf + lane * (k + 2), lane < chunks, k, pair, from, place);
        }
        rank = o != o ? kNoRank : rank_of(o, pair);
        token = rank && rank != kNoRank ? (int32_t)~(uint32_t)pair : -1;
    }
    // the group: every beam's
    unsigned long long* put = a.ranks + (uint64_t)row * 2 * k;
    if (wave == 0 && lane < k) {
        beam_put(put + lane, rank);
        beam_put(put + k + lane, (uint32_t)token);
    }
    if (!beam_last(a.count + (uint64_t)a.groups * a.beams + group, a.beams, &flag)) return;
    const unsigned long long* all = a.ranks + (uint64_t)group * a.beams * 2 * k;
    for (uint32_t i = tid; i < a.beams * 2 * k; i += 256) {
        const uint32_t b = i / (2 * k), j = i - b * 2 * k;
        const unsigned long long x = beam_get(all + i);
        if (j < k) ranks[b * k + j] = x;
        else tokens[b * k + j - k] = (uint32_t)x;
    }
    __syncthreads();
    if (wave != 0) return;
    uint32_t beam, place;
    const bool off = __ballot(lane < a.beams && ranks[lane * k] == kNoRank) != 0;
    merge_lists(ranks + lane * k, lane < a.beams && !off, k, rank, beam, place);
    if (off && lane == 0) report_error(a.err_word, model_key(a.group0 + group, kStOOut, 0));
    if (lane < k) {
        const uint64_t o = (uint64_t)group * k + lane;
        a.out_scores[o] = rank ? (float)rank_value(rank) : -INFINITY;
        a.parents[o] = rank ? (int32_t)beam : -1;
        a.tokens[o] = rank ? (int32_t)tokens[beam * k + place] : -1;
    }
}

// Logits of a thread at a time, and of a workgroup: few rows are cut finer, to fill the CUs (4 rows of 128256
// tokens: 252 workgroups), many into about 512 workgroups (128 rows of 151936: 38.2 us; 768 the same, 1024 39.9,
// 384 42.7); at most 64 chunks, which a wave's lanes merge.
static uint32_t select_unroll(uint64_t rows, uint64_t vocabulary) { return rows * vocabulary <= (1u << 21) ? 2 : 4; }
static uint32_t select_chunk(uint64_t rows, uint64_t vocabulary) {
    const uint64_t unit = 1024 * select_unroll(rows, vocabulary), most = 512 / rows < 1 ? 1 : 512 / rows < 64 ? 512 / rows : 64;
    uint64_t n = (vocabulary + unit - 1) / unit;
    n = n < most ? n : most;
    return (uint32_t)(((vocabulary + n - 1) / n + 3) / 4 * 4);
}
static uint64_t select_chunks(uint64_t rows, uint64_t vocabulary) {
    const uint64_t c = select_chunk(rows, vocabulary);
    return (vocabulary + c - 1) / c;
}
// Groups of a launch (a grid's second dimension has 65535 workgroups), which use the same scratch and counters.
static uint64_t select_groups(const SelectArgs& a) { return a.groups < 65535 / a.beams ? a.groups : 65535 / a.beams; }
// Whether all chunks of a group go through one workgroup's LDS (32 KB at most): one exchange less.
static bool select_once(const SelectArgs& a, uint64_t chunks) {
    return a.beams * chunks <= 256 && a.beams * chunks * (a.best + 2) <= 4096;
}
size_t beam_select_bytes(const SelectArgs& a) {
    const uint64_t chunks = select_chunks((uint64_t)a.groups * a.beams, a.vocabulary);
    const bool once = select_once(a, chunks);
    const uint64_t lists = chunks > 1 || once ? chunks * (a.best + 2) : 0, ranks = once ? 0 : 2 * a.best;
    return select_groups(a) * a.beams * (lists + ranks) * sizeof(unsigned long long);
}
uint64_t beam_select_counters(const SelectArgs& a) { return select_groups(a) * (a.beams + 1); }

hipError_t launch_beam_select(SelectArgs a, void* scratch, hipStream_t s) {
    if (a.groups == 0 || a.groups > 65535 || a.beams == 0 || a.beams > kSelectMaxBeams || a.best == 0 ||
        a.best > kSelectMaxBest || a.vocabulary == 0)
        return hipErrorInvalidValue;
    const uint64_t rows = (uint64_t)a.groups * a.beams, chunks = select_chunks(rows, a.vocabulary), most = select_groups(a);
    a.chunk = select_chunk(rows, a.vocabulary);
    a.once = select_once(a, chunks);
    a.ranks = (unsigned long long*)scratch;
    a.lists = a.ranks + (a.once ? 0 : most * a.beams * 2 * a.best);
    uint64_t words = chunks > 1 ? chunks * (a.best + 2) : 0;
    if (words < 4 * kListMost) words = 4 * kListMost;
    const uint64_t of_beams = ((uint64_t)a.beams * a.best * 3 + 1) / 2;  // (at most 48 KB)
    if (words < of_beams) words = of_beams;
    const uint64_t of_group = a.beams * chunks * (a.best + 2), beside = kSelectMaxBeams + 256 + kFound + kFound / 2;
    if (a.once && words < of_group + beside) words = of_group + beside;
    for (uint64_t g = 0; g < a.groups;) {
        const uint64_t n = a.groups - g < most ? a.groups - g : most;
        SelectArgs p = a;
        p.logits += g * a.beams * a.stride, p.scores += g * a.beams;
        p.out_scores += g * a.best, p.parents += g * a.best, p.tokens += g * a.best;
        p.group0 = (uint32_t)g, p.groups = (uint32_t)n;
        const dim3 grid((uint32_t)chunks, (uint32_t)(n * a.beams)), block(256);
        const size_t lds = words * sizeof(unsigned long long);
        if (select_unroll(rows, a.vocabulary) == 2) hipLaunchKernelGGL(beam_select_kernel<2>, grid, block, lds, s, p);
        else hipLaunchKernelGGL(beam_select_kernel<4>, grid, block, lds, s, p);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        g += n;
    }
    return hipSuccess;
}

}  // namespace rlq
