// kv.hip - a paged KV cache on gfx950: pages off a free list, the store of rotated
// keys and of values, attention of new tokens over the pages, and the beams' tables.
//
// A cache's layer holds, for each page and KV head, a plane of `page` tokens:
// token after token their `dim` values (f32, f16, bf16), or (Q8_0) their levels and
// after those, token after token, the f16 scales of their blocks of 32.
#include "rlq_device.hpp"
#include "rlq_internal.hpp"
#include "rlq_q8k.hpp"

namespace rlq {

// ---------------------------------------------------------------------------
// Pages of the requests
// ---------------------------------------------------------------------------

constexpr uint32_t kPlanThreads = 1024, kPlanPer = kKvMaxRequests / kPlanThreads;

// Why a request gets no pages (rlq.h, RLQ_INVALID_STATE of rlq_kv_pages).
enum PagesRefusal : uint32_t { kBadCount = 0, kNoPage = 1, kNoColumn = 2, kNoRow = 3, kBadLength = 4 };

// The sum over the threads before this one, and over all of them.
__device__ __forceinline__ uint64_t plan_scan(uint64_t v, uint64_t* part, uint64_t& total) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t sum = v;
    for (int m = 1; m < 64; m <<= 1) {
        const uint64_t o = __shfl_up(sum, m, 64);
        if ((int)lane >= m) sum += o;
    }
    __syncthreads();  // (part is free)
    if (lane == 63) part[wave] = sum;
    __syncthreads();
    uint64_t before = 0;
    total = 0;
    for (uint32_t w = 0; w < kPlanThreads / 64; ++w) {
        if (w < wave) before += part[w];
        total += part[w];
    }
    return before + sum - v;
}

// The last of the n + 1 ascending numbers that is not above v (at[0] = 0 <= v < at[n]).
template <class P>
__device__ __forceinline__ uint32_t segment_of(const P* at, uint32_t n, uint32_t v) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if ((uint32_t)at[mid] <= v) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Row t of the batch: its request, position and slot; -1 behind the last.
template <class P>
__device__ __forceinline__ void pages_row(const PagesArgs& a, const P* starts, uint32_t total, uint32_t t, const int32_t* after) {
    int32_t request = -1, position = -1;
    int64_t slot = -1;
    if (t < total) {
        const uint32_t r = segment_of(starts, a.requests, t);
        const uint32_t ahead = (uint32_t)starts[r + 1] - t;  // rows of the request from this one on
        request = (int32_t)r;
        position = after[r] - (int32_t)ahead;
        const int32_t page = a.tables[(uint64_t)r * a.width + ((uint32_t)position >> a.log_page)];
        slot = ((int64_t)page << a.log_page) + (position & ((1 << a.log_page) - 1));
    }
    a.out_requests[t] = request;
    a.positions[t] = position;
    a.slots[t] = slot;
}

// One workgroup: sums over the requests, the ended requests' pages onto the free
// list, pages off its top (request after request, the t-th from the top is the t-th
// page taken), and, where `rows`, the batch's rows.  Everything is checked before
// anything is written.
__global__ __launch_bounds__(1024) void pages_plan_kernel(PagesArgs a, uint32_t rows) {
    __shared__ uint64_t part[kPlanThreads / 64];
    __shared__ uint32_t need[kKvMaxRequests + 1], start[kKvMaxRequests + 1], gone[kKvMaxRequests];
    __shared__ uint16_t ended[kKvMaxRequests];
    __shared__ uint32_t n_ended, first_bad;
    __shared__ unsigned long long bad_page;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.requests;
    const int64_t free0 = *a.count;
    if (tid == 0) n_ended = 0, first_bad = 0xffffffffu, bad_page = ~0ull;
    __syncthreads();

    // a request's columns of the table in use, the pages and the rows it gets
    int32_t before[kPlanPer], more[kPlanPer];
    uint64_t pages = 0, tokens = 0;
    uint32_t refused = 0xffffffffu;  // request * 8 + the reason
    auto refuse = [&](uint32_t r, uint32_t why) { refused = r * 8 + why < refused ? r * 8 + why : refused; };
    auto held = [&](int64_t len) { return (uint64_t)(len + (1 << a.log_page) - 1) >> a.log_page; };
#pragma unroll
    for (uint32_t i = 0; i < kPlanPer; ++i) {
        const uint32_t r = tid * kPlanPer + i;
        before[i] = r < n ? a.before[r] : 0;
        more[i] = r < n ? a.more[r] : 0;
        const int64_t after = (int64_t)before[i] + (more[i] > 0 ? more[i] : 0);
        if (before[i] < 0 || after > 0x7fffffff) {
            refuse(r, kBadLength);
            before[i] = more[i] = 0;
        } else if (held(after) > a.width) {
            refuse(r, kNoColumn);
            before[i] = more[i] = 0;
        }
        if (r < n) {
            gone[r] = 0;
            if (more[i] < 0) ended[atomicAdd(&n_ended, 1u)] = (uint16_t)r;
        }
        if (more[i] > 0) pages += held(after) - held(before[i]), tokens += (uint32_t)more[i];
    }
    __syncthreads();
    for (uint32_t i = wave; i < n_ended; i += kPlanThreads / 64) {  // (a wave per ended request)
        const uint32_t r = ended[i];
        const int32_t* row = a.owned + (uint64_t)r * a.width;
        const uint32_t cols = (uint32_t)held(a.before[r]);
        uint32_t some = 0;
        for (uint32_t c = 0; c < cols; c += 64) {
            const int32_t p = c + lane < cols ? row[c + lane] : -1;
            if (p >= 0 && (uint32_t)p >= a.pages) atomicMin(&bad_page, (unsigned long long)r * a.width + c + lane);
            some += (uint32_t)__builtin_popcountll(__ballot(p >= 0));
        }
        if (lane == 0) gone[r] = some;
    }
    __syncthreads();

    uint64_t total_need, total_gone, total_rows, back = 0;
    uint64_t at_need = plan_scan(pages, part, total_need), at_row = plan_scan(tokens, part, total_rows);
#pragma unroll
    for (uint32_t i = 0; i < kPlanPer; ++i)
        if (tid * kPlanPer + i < n) back += gone[tid * kPlanPer + i];
    uint64_t at_gone = plan_scan(back, part, total_gone);
    const bool sound = free0 >= 0 && free0 <= (int64_t)a.pages && (uint64_t)free0 + total_gone <= a.pages;
    const uint64_t top = (sound ? (uint64_t)free0 : 0) + total_gone;
    if (!sound) refuse(0, kBadCount);
#pragma unroll
    for (uint32_t i = 0; i < kPlanPer; ++i) {
        const uint32_t r = tid * kPlanPer + i;
        if (r >= n) break;
        const int64_t after = (int64_t)before[i] + (more[i] > 0 ? more[i] : 0);
        need[r] = (uint32_t)(at_need < 0xffffffffull ? at_need : 0xffffffffull);
        start[r] = (uint32_t)(at_row < 0xffffffffull ? at_row : 0xffffffffull);
        const uint32_t g = gone[r];
        gone[r] = (uint32_t)(at_gone < 0xffffffffull ? at_gone : 0xffffffffull);
        at_gone += g;
        if (more[i] > 0) at_need += held(after) - held(before[i]), at_row += (uint32_t)more[i];
        if (at_need > top) refuse(r, kNoPage);
        if (at_row > a.tokens) refuse(r, kNoRow);
    }
    if (refused != 0xffffffffu) atomicMin(&first_bad, refused);
    if (tid == 0) need[n] = (uint32_t)total_need, start[n] = (uint32_t)total_rows;  // (not past 32 bits, or refused)
    __syncthreads();
    const bool bad = first_bad != 0xffffffffu || bad_page != ~0ull;
    if (tid == 0) {
        *a.refused = bad;
        if (bad_page != ~0ull) report_error(a.err_word, bounds_key(bad_page));
        else if (bad) report_error(a.err_word, model_key(first_bad / 8, kStPages, first_bad % 8));
    }
    if (bad) return;

    for (uint32_t i = wave; i < n_ended; i += kPlanThreads / 64) {
        const uint32_t r = ended[i], cols = (uint32_t)held(a.before[r]);
        int32_t* row = a.owned + (uint64_t)r * a.width;
        uint64_t to = (uint64_t)free0 + gone[r];
        for (uint32_t c = 0; c < cols; c += 64) {
            const int32_t p = c + lane < cols ? row[c + lane] : -1;
            const unsigned long long m = __ballot(p >= 0);
            if (p >= 0) {
                a.free[to + __builtin_popcountll(m & ((1ull << lane) - 1))] = p;
                row[c + lane] = -1;
            }
            to += __builtin_popcountll(m);
        }
    }
    __syncthreads();
    for (uint32_t t = tid; t < (uint32_t)total_need; t += kPlanThreads) {
        const uint32_t r = segment_of(need, n, t);
        const uint64_t at = (uint64_t)r * a.width + held(a.before[r]) + (t - need[r]);
        const int32_t p = a.free[top - 1 - t];
        a.tables[at] = p;
        if (a.owned != a.tables) a.owned[at] = p;
    }
    __syncthreads();  // (the lengths may take the place of `before`)
#pragma unroll
    for (uint32_t i = 0; i < kPlanPer; ++i) {
        const uint32_t r = tid * kPlanPer + i;
        if (r >= n) break;
        a.after[r] = more[i] < 0 ? 0 : before[i] + more[i];
        a.starts[r] = (int32_t)start[r];
    }
    if (tid == 0) a.starts[n] = (int32_t)total_rows, *a.count_after = (int32_t)(top - total_need);
    if (!rows) return;
    __syncthreads();
    for (uint32_t t = tid; t < a.tokens; t += kPlanThreads) pages_row(a, start, (uint32_t)total_rows, t, a.after);
}

__global__ __launch_bounds__(256) void pages_rows_kernel(PagesArgs a) {
    const uint32_t t = blockIdx.x * 256 + threadIdx.x;
    if (t >= a.tokens || *a.refused) return;
    pages_row(a, a.starts, (uint32_t)a.starts[a.requests], t, a.after);
}

hipError_t launch_kv_pages(const PagesArgs& a, hipStream_t s) {
    if (a.requests == 0 || a.requests > kKvMaxRequests || a.tokens > 0x7fffffffu) return hipErrorInvalidValue;
    const bool one = a.tokens <= 4096;
    hipLaunchKernelGGL(pages_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a, one ? 1u : 0u);
    if (!one) hipLaunchKernelGGL(pages_rows_kernel, dim3((a.tokens + 255) / 256), dim3(256), 0, s, a);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Store
// ---------------------------------------------------------------------------

template <uint32_t T>
__device__ __forceinline__ uint64_t kv_row(uint32_t dim) {  // bytes of a token's values (Q8_0: levels) in a plane
    return T == kQ8_0 ? dim : T == kF32 ? 4 * dim : 2 * dim;
}
template <uint32_t T>
__device__ __forceinline__ uint64_t kv_plane(uint32_t dim, uint32_t log_page) {
    return (T == kQ8_0 ? dim + dim / 16 : kv_row<T>(dim)) << log_page;
}

__device__ __forceinline__ uint32_t bf16_bits(float v) {  // ties to even; v is finite
    const uint32_t b = __float_as_uint(v);
    return (b + 0x7fffu + ((b >> 16) & 1)) >> 16;
}

// A token's query, key and value heads, dim / 4 lanes a head and four values a lane.
// The first 2 * half values of a query or key head are rotated:
//   (x, y) -> (x cos a - y sin a, x sin a + y cos a),  a = position * freq[i]
// of neighbours (pairs) or of values half apart; angle, sine, cosine, products and sum in
// f64, rounded once to f32, so that the stored 16 bits and levels are defined to the last
// one.  A wave loads whole heads before it stores them: q_out may be q.
template <uint32_t T>
__global__ __launch_bounds__(256) void kv_store_kernel(StoreArgs a) {
    __shared__ double2 turn[128];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, dim = a.c.dim;
    const uint64_t t = blockIdx.x;
    const int64_t slot = a.slots[t];
    if (slot == -1) return;  // a row behind the batch's last
    if (slot < 0 || (uint64_t)slot >= a.c.pages << a.c.log_page) {
        if (threadIdx.x == 0) report_error(a.err_word, bounds_key(t));
        return;
    }
    if (threadIdx.x < a.half) {
        double s, c;
        sincos((double)a.positions[t] * (double)a.freqs[threadIdx.x], &s, &c);
        turn[threadIdx.x] = make_double2(c, s);
    }
    __syncthreads();
    const uint32_t L = dim / 4, per = 64 / L, group = lane / L, e = 4 * (lane % L);
    const uint32_t kv = a.c.kv_heads, heads = a.heads + 2 * kv;
    const uint64_t page = (uint64_t)slot >> a.c.log_page, row = (uint64_t)slot & ((1u << a.c.log_page) - 1);

    // four values of head h, and whether one is not finite
    auto values = [&](uint32_t h, float (&y)[4]) {
        const bool q = h < a.heads, k = !q && h < a.heads + kv;
        const float* x = q ? a.q + t * a.q_stride + (uint64_t)h * dim
                           : k ? a.k + t * a.k_stride + (uint64_t)(h - a.heads) * dim
                               : a.v + t * a.v_stride + (uint64_t)(h - a.heads - kv) * dim;
        bool off = false;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const uint32_t i = e + j;
            y[j] = x[i];
            if ((q || k) && i < 2 * a.half) {
                const bool second = a.pairs ? i & 1 : i >= a.half;
                const uint32_t other = a.pairs ? i ^ 1 : second ? i - a.half : i + a.half;
                const double2 cs = turn[a.pairs ? i / 2 : second ? i - a.half : i];
                const double m = (double)y[j] * cs.x, o = (double)x[other] * cs.y;
                y[j] = (float)(second ? o + m : m - o);
            }
            off |= !finite(y[j]);
            if (T == kF16 && !q) off |= !finite((float)(_Float16)y[j]);
            if (T == kBF16 && !q) off |= !finite(__uint_as_float(bf16_bits(y[j]) << 16));
        }
        return off;
    };

    int bad = 0;
    for (uint32_t h = wave * per + group; h < heads && group < per; h += 4 * per) {
        float y[4];
        if (values(h, y)) {
            bad = 1;
            report_error(a.err_word, error_key(t, kKindNonFinite, (uint64_t)h * dim + e));
        } else if (T == kQ8_0 && h >= a.heads && norm_q8_0(y).bad) {
            bad = 1;
            report_error(a.err_word, error_key(t, kKindScale, ((uint64_t)(h - a.heads) * dim + e) / 32));
        }
    }
    if (__syncthreads_or(bad)) return;
    for (uint32_t h = wave * per + group; h < heads && group < per; h += 4 * per) {
        float y[4];
        values(h, y);
        if (h < a.heads) {
            float* out = a.q_out + t * a.out_stride + (uint64_t)h * dim + e;
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) out[j] = y[j];
            continue;
        }
        const uint32_t g = h - a.heads < kv ? h - a.heads : h - a.heads - kv;
        uint8_t* plane = (h - a.heads < kv ? a.c.k + page * a.c.k_stride : a.c.v + page * a.c.v_stride) +
                         g * kv_plane<T>(dim, a.c.log_page);
        uint8_t* to = plane + row * kv_row<T>(dim);
        if constexpr (T == kF32) {
            *(float4*)(to + 4 * e) = make_float4(y[0], y[1], y[2], y[3]);
        } else if constexpr (T == kQ8_0) {
            const NormQ q = norm_q8_0(y);
            *(uint32_t*)(to + e) = q.q;
            if (e % 32 == 0)
                *(uint16_t*)(plane + ((uint64_t)dim << a.c.log_page) + 2 * (row * (dim / 32) + e / 32)) =
                    (uint16_t)float_to_half_bits(q.d);
        } else {
            uint32_t b[4];
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)
                b[j] = T == kF16 ? (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)y[j]) : bf16_bits(y[j]);
            *(uint2*)(to + 2 * e) = make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
        }
    }
}

hipError_t launch_kv_store(const StoreArgs& a, hipStream_t s) {
    if (a.tokens == 0 || a.tokens > 0x7fffffffu || a.c.dim % 32 || a.c.dim > 256 || 2 * a.half > a.c.dim)
        return hipErrorInvalidValue;
    const dim3 grid((uint32_t)a.tokens), block(256);
    switch (a.c.type) {
        case kF32: hipLaunchKernelGGL(kv_store_kernel<kF32>, grid, block, 0, s, a); break;
        case kF16: hipLaunchKernelGGL(kv_store_kernel<kF16>, grid, block, 0, s, a); break;
        case kBF16: hipLaunchKernelGGL(kv_store_kernel<kBF16>, grid, block, 0, s, a); break;
        case kQ8_0: hipLaunchKernelGGL(kv_store_kernel<kQ8_0>, grid, block, 0, s, a); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------

// Four values of a token from element e on.
template <uint32_t T>
__device__ __forceinline__ float4 kv_load4(const uint8_t* plane, uint32_t row, uint32_t e, uint32_t dim, uint32_t log_page) {
    const uint8_t* p = plane + row * kv_row<T>(dim);
    if constexpr (T == kF32) {
        return *(const float4*)(p + 4 * e);
    } else if constexpr (T == kQ8_0) {
        const uint32_t q = *(const uint32_t*)(p + e);
        const float d = half_to_float(*(const uint16_t*)(plane + ((uint64_t)dim << log_page) + 2 * (row * (dim / 32) + e / 32)));
        return make_float4((float)(int8_t)q * d, (float)(int8_t)(q >> 8) * d, (float)(int8_t)(q >> 16) * d,
                           (float)(int8_t)(q >> 24) * d);
    } else {
        const uint2 b = *(const uint2*)(p + 2 * e);
        if constexpr (T == kF16)
            return make_float4(half_to_float(b.x), half_to_float(b.x >> 16), half_to_float(b.y), half_to_float(b.y >> 16));
        return make_float4(__uint_as_float(b.x << 16), __uint_as_float(b.x & 0xffff0000u), __uint_as_float(b.y << 16),
                           __uint_as_float(b.y & 0xffff0000u));
    }
}

// One query head of a row per workgroup: 256 tokens at a time, a thread a token for
// the scores and a thread a value for the output, with a running maximum and sum.
template <uint32_t T>
__global__ __launch_bounds__(256) void kv_attention_kernel(AttnArgs a) {
    __shared__ __align__(16) float q[256], p[256];
    __shared__ int32_t ids[256];
    __shared__ float red[8];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, dim = a.c.dim, row = blockIdx.x, head = blockIdx.y;
    const uint32_t kvh = head / (a.heads / a.c.kv_heads), mask = (1u << a.c.log_page) - 1;
    const int32_t request = a.requests ? a.requests[row] : (int32_t)row;
    if (request == -1) return;  // a row behind the batch's last
    const int32_t last = a.positions[row];
    if (request < 0 || (uint32_t)request >= a.table_rows || last < -1 || last >= (int64_t)a.width << a.c.log_page) {
        if (tid == 0) report_error(a.err_word, bounds_key(row));
        return;
    }
    const int32_t first = a.window && (uint32_t)last + 1 > a.window ? last + 1 - (int32_t)a.window : 0;
    const int32_t* table = a.tables + (uint64_t)request * a.width;
    if (tid < dim) q[tid] = a.q[row * a.q_stride + (uint64_t)head * dim + tid];
    float m = -INFINITY, sum = 0.0f, acc = 0.0f;
    bool lost = false;
    const uint64_t plane = kvh * kv_plane<T>(dim, a.c.log_page);
    for (int64_t base = first; base <= last; base += 256) {
        const int64_t tok = base + tid;
        __syncthreads();  // (p and ids are free, q is there)
        float s = -INFINITY;
        if (tok <= last) {
            int32_t id = table[tok >> a.c.log_page];
            if (id < 0 || (uint64_t)id >= a.c.pages) lost = true, id = 0;
            ids[tid] = id;
            const uint8_t* kp = a.c.k + (uint64_t)id * a.c.k_stride + plane;
            float d = 0.0f;
            for (uint32_t e = 0; e < dim; e += 4) {
                const float4 k = kv_load4<T>(kp, (uint32_t)tok & mask, e, dim, a.c.log_page);
                d = __builtin_fmaf(k.x, q[e], d);
                d = __builtin_fmaf(k.y, q[e + 1], d);
                d = __builtin_fmaf(k.z, q[e + 2], d);
                d = __builtin_fmaf(k.w, q[e + 3], d);
            }
            s = d * a.scale;
        }
        const float w = wave_max(s);
        if (lane == 0) red[wave] = w;
        __syncthreads();
        const float top = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        const float e = tok <= last ? expf(s - top) : 0.0f, shrink = m == -INFINITY ? 0.0f : expf(m - top);
        p[tid] = e;
        const float part = wave_sum(e);
        if (lane == 0) red[4 + wave] = part;
        __syncthreads();
        sum = sum * shrink + ((red[4] + red[5]) + (red[6] + red[7]));
        acc = acc * shrink;
        m = top;
        if (tid < dim) {
            const uint32_t n = last - base + 1 < 256 ? (uint32_t)(last - base + 1) : 256;
            for (uint32_t j = 0; j < n; ++j) {
                const uint8_t* vp = a.c.v + (uint64_t)ids[j] * a.c.v_stride + plane;
                const float4 v = kv_load4<T>(vp, (uint32_t)(base + j) & mask, tid & ~3u, dim, a.c.log_page);
                const float one = (tid & 2) ? (tid & 1 ? v.w : v.z) : (tid & 1 ? v.y : v.x);
                acc = __builtin_fmaf(p[j], one, acc);
            }
        }
        __syncthreads();
    }
    const float y = last < 0 ? 0.0f : acc / sum;
    const bool off = tid < dim && !finite(y);
    if (__syncthreads_or(lost)) {
        if (tid == 0) report_error(a.err_word, bounds_key(row));
        return;
    }
    if (__syncthreads_or(off)) {
        if (tid == 0) report_error(a.err_word, model_key(row, kStAttnOut, 0));
        return;
    }
    if (tid < dim) a.out[row * a.out_stride + (uint64_t)head * dim + tid] = y;
}

hipError_t launch_kv_attention(const AttnArgs& a, hipStream_t s) {
    if (a.rows == 0 || a.rows > 65535 || a.heads == 0 || a.heads > 65535 || a.c.dim % 32 || a.c.dim > 256)
        return hipErrorInvalidValue;
    const dim3 grid(a.rows, a.heads), block(256);
    switch (a.c.type) {
        case kF32: hipLaunchKernelGGL(kv_attention_kernel<kF32>, grid, block, 0, s, a); break;
        case kF16: hipLaunchKernelGGL(kv_attention_kernel<kF16>, grid, block, 0, s, a); break;
        case kBF16: hipLaunchKernelGGL(kv_attention_kernel<kBF16>, grid, block, 0, s, a); break;
        case kQ8_0: hipLaunchKernelGGL(kv_attention_kernel<kQ8_0>, grid, block, 0, s, a); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// The beams' tables
// ---------------------------------------------------------------------------

// A group's beams after a choice: beam b goes on from parents[b] (-1: from itself).
// Whole pages are shared: their columns of the tables are the parent's.  The page that
// is being filled is each beam's own: its first tokens are copied, in every tensor.
// A thread takes one column, or one piece at one place of all beams' pages: it has
// loaded all before it stores any, so the beams may change places among themselves.
//
// grid: pieces (or columns), groups, tensors (the tables first).
template <int MB>
__global__ __launch_bounds__(256) void beam_reorder_kernel(ReorderArgs a) {
    __shared__ int32_t from[MB], source[MB], mine[MB];
    __shared__ uint32_t tail_s, rows_s;
    const uint32_t tid = threadIdx.x, g = blockIdx.y, B = a.beams;
    const uint64_t beam0 = (uint64_t)g * B;
    uint64_t wrong = ~0ull;
    if (tid < B) {
        const int32_t p = a.parents[beam0 + tid], len = a.lengths[beam0 + tid];
        from[tid] = p == -1 ? (int32_t)tid : p;
        const uint64_t tail = (uint64_t)(len < 0 ? 0 : len) >> a.log_page;
        const uint32_t rows = len & ((1 << a.log_page) - 1);
        if (p < -1 || p >= (int32_t)B || len < 0 || len != a.lengths[beam0] || tail + (rows > 0) > a.width) wrong = beam0 + tid;
        else if (rows) {
            mine[tid] = a.tables[(beam0 + tid) * a.width + tail];
            if (mine[tid] < 0 || (uint64_t)mine[tid] >= a.pages) wrong = beam0 + tid;
        }
        if (tid == 0) tail_s = (uint32_t)tail, rows_s = rows;
    }
    if (__syncthreads_or(wrong != ~0ull)) {  // (every workgroup of the group finds the same)
        if (wrong != ~0ull) report_error(a.err_word, bounds_key(wrong));
        return;
    }
    if (tid < B) source[tid] = mine[from[tid]];
    __syncthreads();
    const uint32_t tail = tail_s, rows = rows_s;
    if (blockIdx.z == 0) {
        if (!a.last) return;  // (the tables are taken over by the last launch)
        for (uint32_t c = blockIdx.x * 256 + tid; c < tail; c += gridDim.x * 256) {
            int32_t v[MB];
#pragma unroll
            for (int b = 0; b < MB; ++b)
                if (b < (int)B) v[b] = a.tables[(beam0 + from[b]) * a.width + c];
#pragma unroll
            for (int b = 0; b < MB; ++b)
                if (b < (int)B && from[b] != b) a.tables[(beam0 + b) * a.width + c] = v[b];
        }
        return;
    }
    if (!rows) return;
    uint8_t* base = a.tensors[blockIdx.z - 1];
    const uint64_t stride = (blockIdx.z - 1) & 1 ? a.v_stride : a.k_stride;
    // a plane's rows in use, as pieces of 16 bytes; Q8_0: and the scales' in pieces of 2
    const uint32_t pieces = rows * a.row_bytes / 16, scales = rows * a.scale_bytes / 2, all = pieces + scales;
    const uint32_t plane = (a.row_bytes + a.scale_bytes) << a.log_page;
    const uint64_t n = (uint64_t)a.kv_heads * all;
    for (uint64_t i = blockIdx.x * 256ull + tid; i < n; i += gridDim.x * 256ull) {
        const uint32_t h = (uint32_t)(i / all), r = (uint32_t)(i - (uint64_t)h * all);
        const uint64_t at = (uint64_t)h * plane;
        if (r < pieces) {
            uint4 v[MB];
#pragma unroll
            for (int b = 0; b < MB; ++b)
                if (b < (int)B && from[b] != b) v[b] = *(const uint4*)(base + (uint64_t)source[b] * stride + at + 16 * r);
#pragma unroll
            for (int b = 0; b < MB; ++b)
                if (b < (int)B && from[b] != b) *(uint4*)(base + (uint64_t)mine[b] * stride + at + 16 * r) = v[b];
        } else {
            const uint64_t o = at + ((uint64_t)a.row_bytes << a.log_page) + 2 * (r - pieces);
            uint16_t v[MB];
#pragma unroll
            for (int b = 0; b < MB; ++b)
                if (b < (int)B && from[b] != b) v[b] = *(const uint16_t*)(base + (uint64_t)source[b] * stride + o);
#pragma unroll
            for (int b = 0; b < MB; ++b)
                if (b < (int)B && from[b] != b) *(uint16_t*)(base + (uint64_t)mine[b] * stride + o) = v[b];
        }
    }
}

hipError_t launch_beam_reorder(const ReorderArgs& a, hipStream_t s) {
    if (a.groups == 0 || a.groups > 65535 || a.beams == 0 || a.beams > kReorderMaxBeams || a.n_tensors > 2 * kReorderLayers)
        return hipErrorInvalidValue;
    const uint64_t pieces = (uint64_t)a.kv_heads * (a.row_bytes / 16 + a.scale_bytes / 2) << a.log_page;
    uint64_t x = (pieces + 255) / 256;
    x = x < 1 ? 1 : x > 1024 ? 1024 : x;
    const dim3 grid((uint32_t)x, a.groups, 1 + a.n_tensors), block(256);
    if (a.beams <= 4) hipLaunchKernelGGL(beam_reorder_kernel<4>, grid, block, 0, s, a);
    else if (a.beams <= 8) hipLaunchKernelGGL(beam_reorder_kernel<8>, grid, block, 0, s, a);
    else if (a.beams <= 16) hipLaunchKernelGGL(beam_reorder_kernel<16>, grid, block, 0, s, a);
    else hipLaunchKernelGGL(beam_reorder_kernel<kReorderMaxBeams>, grid, block, 0, s, a);
    return hipGetLastError();
}

}  // namespace rlq
