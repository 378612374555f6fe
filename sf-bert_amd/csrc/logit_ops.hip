// Operators on rows of logits: the log probabilities of given tokens with entropy and top alternatives, and the
// distillation loss against a teacher's top logits, each with its gradient.  No counterpart in the reference, whose
// only loss is softmax_cross_entropy_with_logits (ewops.h:233-261).
//
// With s = scale, c = s log2(e), a row x and any reference m:  S = sum_j 2^((x_j - m) c),  l = log2 S,
//   ln p_j = (x_j - m) s - ln2 l,   entropy = ln2 (l - W / S) with W = sum_j 2^t_j t_j, t_j = (x_j - m) c.
// Everything is held in fp32.  The row is read once; (m, l) is what the backward pass is given.
#include "common.hip.h"

namespace sfb {

constexpr uint32_t kMaxTop = 64;      // alternatives per row
constexpr uint32_t kMaxSlots = 256;   // given tokens, or entries of a teacher's list, per row
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kInf = __builtin_inff();
// Scaled reference (m c) of a lane that has not met a logit yet; logits whose scaled value passes kWide in either
// direction are left to a second pass over the row that subtracts the maximum before it scales.
constexpr float kNoReference = -1.0e30f;
constexpr float kWide = 1.0e29f;

// A 16-byte vector of logits.
template <typename T> struct LogitVec;
template <> struct LogitVec<float> {
    static constexpr int N = 4;
    __device__ static __forceinline__ void unpack(u32x4 raw, float (&v)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t bits = raw[i];   // (a bit cast of a vector's element itself reads its first one)
            v[i] = __builtin_bit_cast(float, bits);
        }
    }
    __device__ static __forceinline__ u32x4 pack(const float (&v)[N]) {
        u32x4 r;
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = __builtin_bit_cast(uint32_t, v[i]);
        return r;
    }
    __device__ static __forceinline__ float load(const float* p) { return *p; }
    __device__ static __forceinline__ void store(float* p, float v) { *p = v; }
};
template <> struct LogitVec<__bf16> {
    static constexpr int N = 8;
    __device__ static __forceinline__ void unpack(u32x4 raw, float (&v)[N]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __builtin_bit_cast(float, raw[i] << 16);
            v[2 * i + 1] = __builtin_bit_cast(float, raw[i] & 0xffff0000u);
        }
    }
    __device__ static __forceinline__ u32x4 pack(const float (&v)[N]) {
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
        return r;
    }
    __device__ static __forceinline__ float load(const __bf16* p) { return bf16_bits_to_f32(*(const uint16_t*)p); }
    __device__ static __forceinline__ void store(__bf16* p, float v) { *(uint16_t*)p = (uint16_t)pack_bf16(v, 0.f); }
};

// A row as whole 16-byte vectors and the elements before and after them: rows start at any element (odd vocabularies).
template <typename T> struct RowSpan {
    const T* row;
    uint32_t head, vecs, tail;
    __device__ __forceinline__ RowSpan(const T* r, uint32_t vocab) : row(r) {
        constexpr uint32_t N = LogitVec<T>::N;
        const uint32_t at = (uint32_t)((uintptr_t)r & 15u) / sizeof(T);
        head = at ? N - at : 0;
        if (head > vocab) head = vocab;
        vecs = (vocab - head) / N;
        tail = vocab - head - vecs * N;
    }
    // element index of the edge element thread t takes care of (one each), or -1
    __device__ __forceinline__ int32_t edge(uint32_t t) const {
        if (t < head) return (int32_t)t;
        if (t < head + tail) return (int32_t)(head + vecs * LogitVec<T>::N + (t - head));
        return -1;
    }
    __device__ __forceinline__ u32x4 vec(uint32_t i) const { return *(const u32x4*)(row + head + (size_t)i * LogitVec<T>::N); }
    __device__ __forceinline__ uint32_t index(uint32_t i) const { return head + i * LogitVec<T>::N; }
};

// What a lane knows of its part of a row: sum and dot are relative to the scaled reference ref2, which lags the
// running maximum by at most kLazyRescaleLog2 powers of two, so that it hardly ever moves after the first vector.
struct RowSum {
    float ref, ref2;   // reference logit and fl(ref c)
    float top;         // largest logit (NaN left out)
    float sum, dot;    // sum 2^t, sum 2^t t with t = x c - ref2
    __device__ __forceinline__ void clear() { ref = top = -kInf; ref2 = kNoReference; sum = dot = 0.f; }

    // 2^t t with t = -inf standing for 0 (a masked logit); a NaN reaches both sums through 2^t
    template <bool ENTROPY, int N>
    __device__ __forceinline__ void add(const float (&v)[N], float c) {
        float hi = v[0];
#pragma unroll
        for (int i = 1; i < N; ++i) hi = fmaxf(hi, v[i]);
        top = fmaxf(top, hi);
        const float hi2 = hi * c;
        if (hi2 > ref2 + kLazyRescaleLog2) {
            const float d = ref2 - hi2, f = exp2_fast(d);
            if (ENTROPY) dot = f * (dot + fmaxf(d, -256.f) * sum);
            sum *= f;
            ref = hi;
            ref2 = hi2;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float t = fmaf(v[i], c, -ref2), e = exp2_fast(t);
            sum += e;
            if (ENTROPY) dot = fmaf(e, fmaxf(t, -256.f), dot);
        }
    }
    // the same relative to a given reference, subtracted before scaling
    template <bool ENTROPY, int N>
    __device__ __forceinline__ void add_wide(const float (&v)[N], float c, float m) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float t = (v[i] - m) * c, e = exp2_fast(t);
            sum += e;
            if (ENTROPY) dot = fmaf(e, fmaxf(t, -256.f), dot);
        }
    }
    // from relative to fl(ref c) to relative to ref c: the reference of different lanes, and of the backward pass, is
    // the logit itself
    template <bool ENTROPY> __device__ __forceinline__ void settle(float c) {
        if (ref == -kInf) return;
        const float d = fmaf(ref, c, -ref2), f = exp2_fast(-d);
        if (ENTROPY) dot = f * (dot - d * sum);
        sum *= f;
    }
    // to a reference m >= ref
    template <bool ENTROPY> __device__ __forceinline__ void move(float m, float c) {
        const float d = ref == m ? 0.f : (ref - m) * c, f = exp2_fast(d);
        if (ENTROPY) dot = f * (dot + fmaxf(d, -256.f) * sum);
        sum *= f;
        ref = m;
    }
};

template <int THREADS> __device__ __forceinline__ float group_max(float v, float* red) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    if (THREADS == 64) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) v = fmaxf(v, red[w]);
    return v;
}
// sums in an order that depends on nothing but THREADS
template <int THREADS> __device__ __forceinline__ float group_sum(float v, float* red) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
    if (THREADS == 64) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) v += red[w];
    return v;
}

// Order of the alternatives as whole numbers: larger logits first, -0 as +0, NaN above everything; 0 is below every
// logit.  A composite's low word is the complement of the index: of equal logits the lowest index comes first.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
    if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t order) {
    return __builtin_bit_cast(float, order & 0x80000000u ? (order == 0xffffffffu ? 0x7fc00000u : order & 0x7fffffffu) : ~order);
}
__device__ __forceinline__ uint64_t composite(uint32_t order, uint32_t index) { return ((uint64_t)order << 32) | (uint32_t)~index; }

// The k largest of a row whose threads know the largest logit each of them has met.  The k-th largest of those is at
// most the row's k-th largest logit, and about k logits reach it (with 256 threads and k = 20: about 21), so the row
// itself is only read again where a thread's largest does: a handful of vectors.  Rows with more equal or clustered
// logits than the list holds take the exact threshold from counts over the whole row instead.
template <typename T, int THREADS> struct TopSelect {
    static constexpr int LIST = 512;
    static constexpr int N = LogitVec<T>::N;
    uint64_t* list;       // [LIST] in shared memory
    uint32_t* words;      // [THREADS] in shared memory
    uint32_t* count;      // in shared memory

    __device__ __forceinline__ void append(uint32_t order, uint32_t index) {
        const uint32_t at = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        if (at < (uint32_t)LIST) list[at] = composite(order, index);
    }

    // the largest threshold reached by at least k of the threads' largest logits; *exact: it is one of them
    __device__ uint32_t threshold(uint32_t mine, uint32_t k, bool* exact) {
        const uint32_t t = threadIdx.x, lane = t & 63;
        __syncthreads();
        words[t] = mine;
        __syncthreads();
        uint32_t own[THREADS / 64];
#pragma unroll
        for (int i = 0; i < THREADS / 64; ++i) own[i] = words[i * 64 + lane];
        uint32_t limit = 0;
        bool all = true;
        for (int bit = 31; bit >= 0; --bit) {   // every wave does the same
            const uint32_t next = limit | (1u << bit);
            uint32_t n = 0;
#pragma unroll
            for (int i = 0; i < THREADS / 64; ++i) n += (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(own[i] >= next));
            if (n >= k) limit = next;
            if (n == k) { all = false; break; }
        }
        *exact = all;
        return limit;
    }

    // appends the row's logits above (strict) or from `limit` on, reading only where a thread's largest reaches it
    __device__ void collect(const RowSpan<T>& span, uint32_t v0, uint32_t v1, int32_t edge, uint32_t mine, uint32_t limit,
                            bool strict) {
        const uint32_t t = threadIdx.x;
        __shared__ uint32_t n_threads;
        __syncthreads();
        if (t == 0) { *count = 0; n_threads = 0; }
        __syncthreads();
        const bool reached = strict ? mine > limit : mine >= limit;
        if (reached) words[__hip_atomic_fetch_add(&n_threads, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP)] = t;
        __syncthreads();
        const uint32_t each = (v1 - v0 + THREADS - 1) / THREADS, work = n_threads * each;
        for (uint32_t i = t; i < work; i += THREADS) {
            const uint32_t v = v0 + words[i / each] + (i % each) * THREADS;
            if (v < v1) {
                float x[N];
                LogitVec<T>::unpack(span.vec(v), x);
#pragma unroll
                for (int u = 0; u < N; ++u) {
                    const uint32_t o = order_of(x[u]);
                    if (strict ? o > limit : o >= limit) append(o, span.index(v) + u);
                }
            }
            if (*(volatile uint32_t*)count > (uint32_t)LIST) break;
        }
        if (reached && edge >= 0) {
            const uint32_t o = order_of(LogitVec<T>::load(span.row + edge));
            if (strict ? o > limit : o >= limit) append(o, (uint32_t)edge);
        }
        __syncthreads();
    }

    // logits of the row that reach `limit`
    __device__ uint32_t reaching(const RowSpan<T>& span, uint32_t v0, uint32_t v1, int32_t edge, uint32_t limit) {
        uint32_t n = 0;
        for (uint32_t v = v0 + threadIdx.x; v < v1; v += THREADS) {
            float x[N];
            LogitVec<T>::unpack(span.vec(v), x);
#pragma unroll
            for (int u = 0; u < N; ++u) n += order_of(x[u]) >= limit;
        }
        if (edge >= 0) n += order_of(LogitVec<T>::load(span.row + edge)) >= limit;
        __syncthreads();
        if (threadIdx.x == 0) *count = 0;
        __syncthreads();
        if (n) __hip_atomic_fetch_add(count, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        __syncthreads();
        return *count;
    }

    // appends the `want` lowest-index logits equal to `limit`: groups of consecutive elements in rising order, until
    // there are enough
    __device__ void collect_equal(const RowSpan<T>& span, uint32_t vocab, uint32_t limit, uint32_t want) {
        const uint32_t t = threadIdx.x, lane = t & 63;
        uint32_t have = 0;
        for (uint32_t j0 = 0; j0 < vocab && have < want; j0 += THREADS) {
            const uint32_t j = j0 + t;
            const bool equal = j < vocab && order_of(LogitVec<T>::load(span.row + j)) == limit;
            const uint64_t in_wave = __builtin_amdgcn_ballot_w64(equal);
            __syncthreads();
            if (lane == 0) words[t >> 6] = (uint32_t)__builtin_popcountll(in_wave);
            __syncthreads();
            uint32_t at = have + (uint32_t)__builtin_popcountll(in_wave & ((1ull << lane) - 1));
            for (uint32_t w = 0; w < THREADS / 64; ++w) {
                if (w < (t >> 6)) at += words[w];
                have += words[w];
            }
            if (equal && at < want) list[*count + at] = composite(limit, j);
        }
        __syncthreads();
        if (t == 0) *count += want;
        __syncthreads();
    }

    // leaves at least the k largest of the row, as composites, in list[0 .. *count).  top: the thread's largest logit,
    // any: it has one; nan: the row holds NaN (which the threads' largest leave out)
    __device__ void select(const RowSpan<T>& span, uint32_t vocab, int32_t edge, float top, bool any, bool nan, uint32_t k) {
        const uint32_t v0 = 0, v1 = span.vecs;
        const uint32_t mine = nan ? 0xffffffffu : any ? order_of(top) : 0u;
        bool few = false;
        uint32_t limit = 0;
        if (!nan) {
            bool exact;
            limit = threshold(mine, k, &exact);
            collect(span, v0, v1, edge, mine, limit, false);
            if (*count <= (uint32_t)LIST) return;
            if (exact) {   // mostly one value (a masked vocabulary): the k-th largest if fewer than k are above it
                collect(span, v0, v1, edge, mine, limit, true);
                few = *count < k;
            }
        }
        if (!few) {
            limit = 0;
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t next = limit | (1u << bit);
                if (reaching(span, v0, v1, edge, next) >= k) limit = next;
            }
            collect(span, v0, v1, edge, mine, limit, true);
        }
        collect_equal(span, vocab, limit, k - *count);
    }
};

struct LogprobParams {
    const void* logits;
    const int32_t* tokens;
    float *logprob, *entropy, *stats, *top_logprobs;
    int32_t* top_ids;
    uint64_t stride;
    uint32_t vocab, n_tokens, top_k;
    float scale, c;
};

// ln p of a logit x from a row's statistics; a row without any logit above -inf gives -inf
__device__ __forceinline__ float log_prob(float x, float m, float l, float scale) {
    return l == -kInf ? -kInf : (x - m) * scale - l * kLn2;
}

// Sums a row over the work-group's threads: every thread returns with m, sum, dot of the whole row (and its own top).
template <typename T, int THREADS, bool ENTROPY>
__device__ __forceinline__ RowSum sum_row(const RowSpan<T>& span, int32_t edge, float c, float* red) {
    constexpr int N = LogitVec<T>::N;
    constexpr int UNROLL = 4;
    const uint32_t t = threadIdx.x;
    RowSum acc;
    acc.clear();
    float single[1] = {-kInf};
    if (edge >= 0) single[0] = LogitVec<T>::load(span.row + edge);
    for (uint32_t v = t; v < span.vecs; v += THREADS * UNROLL) {
        u32x4 raw[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (v + u * THREADS < span.vecs) raw[u] = span.vec(v + u * THREADS);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (v + u * THREADS < span.vecs) {
                float x[N];
                LogitVec<T>::unpack(raw[u], x);
                acc.template add<ENTROPY>(x, c);
            }
    }
    if (edge >= 0) acc.template add<ENTROPY>(single, c);
    const float top = group_max<THREADS>(acc.top, red);
    if (fabsf(top * c) > kWide && fabsf(top) < kInf) {
        // logits as large as a type's lowest value (masks made of it): the largest is the reference
        acc.sum = acc.dot = 0.f;
        for (uint32_t v = t; v < span.vecs; v += THREADS) {
            float x[N];
            LogitVec<T>::unpack(span.vec(v), x);
            acc.template add_wide<ENTROPY>(x, c, top);
        }
        if (edge >= 0) acc.template add_wide<ENTROPY>(single, c, top);
        acc.ref = top;
    } else {
        acc.template settle<ENTROPY>(c);
        acc.template move<ENTROPY>(group_max<THREADS>(acc.ref, red), c);
    }
    acc.sum = group_sum<THREADS>(acc.sum, red);
    if (ENTROPY) acc.dot = group_sum<THREADS>(acc.dot, red);
    return acc;
}

// One work-group per row.
template <typename T, int THREADS, bool ENTROPY>
__global__ __launch_bounds__(THREADS) void token_logprobs_kernel(LogprobParams p) {
    __shared__ float red[16];
    __shared__ uint64_t list[512];
    __shared__ uint32_t words[THREADS];
    __shared__ uint32_t count;
    const uint32_t t = threadIdx.x;
    const size_t row = blockIdx.x;
    const RowSpan<T> span((const T*)p.logits + row * p.stride, p.vocab);
    const int32_t edge = span.edge(t);
    const RowSum acc = sum_row<T, THREADS, ENTROPY>(span, edge, p.c, red);
    const float m = acc.ref, l = log2f(acc.sum);
    if (t == 0) {
        if (p.stats) { p.stats[2 * row] = m; p.stats[2 * row + 1] = l; }
        if (ENTROPY) {
            const float h = (l - acc.dot / acc.sum) * kLn2;
            p.entropy[row] = l == -kInf || h < 0.f ? 0.f : h;   // (rounding can leave a certain row below zero)
        }
    }
    for (uint32_t i = t; i < p.n_tokens; i += THREADS) {
        const int32_t id = p.tokens[row * p.n_tokens + i];
        float lp = 0.f;
        if (id >= 0 && (uint32_t)id < p.vocab) lp = log_prob(LogitVec<T>::load(span.row + id), m, l, p.scale);
        p.logprob[row * p.n_tokens + i] = lp;
    }
    if (p.top_k == 0) return;
    TopSelect<T, THREADS> top{list, words, &count};
    top.select(span, p.vocab, edge, acc.top, t < span.vecs || edge >= 0, acc.sum != acc.sum, p.top_k);
    const uint32_t n = count;
    for (uint32_t i = t; i < n; i += THREADS) {
        const uint64_t mine = list[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < n; ++j) rank += list[j] > mine;
        if (rank < p.top_k) {
            p.top_ids[row * p.top_k + rank] = (int32_t)~(uint32_t)mine;
            p.top_logprobs[row * p.top_k + rank] = log_prob(logit_of((uint32_t)(mine >> 32)), m, l, p.scale);
        }
    }
}

// ---- gradients ------------------------------------------------------------------------------------------------
// Both operators' gradients have one form.  With coefficients c_i on tokens id_i, C = sum_i c_i over the valid ones and
// g the gradient of the entropy H:   dx_j = s ( sum_{i: id_i = j} c_i - C p_j - g p_j (ln p_j + H) ).
struct GradParams {
    const void* logits;
    void* d_logits;
    const int32_t* ids;      // [rows][n]
    const float* stats;
    const float *entropy, *d_entropy;   // or NULL
    const float* d_logprob;  // coefficients [rows][n] ...
    const void* teacher;     // ... or a teacher's logits [rows][n] and
    const float* d_loss;     // the gradient of each row's loss
    uint64_t stride;
    uint32_t vocab, n, chunks, chunk_vecs;
    int teacher_bf16;
    float scale, c;
};

__device__ __forceinline__ float teacher_logit(const void* z, int as_bf16, size_t i) {
    return as_bf16 ? bf16_bits_to_f32(((const uint16_t*)z)[i]) : ((const float*)z)[i];
}

// Softmax of a teacher's list over its valid slots, by one wave: q[0 .. n) and returns sum q log2 q; *some: there is a
// distribution (a valid slot above -inf).
__device__ __forceinline__ float teacher_softmax(const int32_t* ids, const void* z, int as_bf16, size_t first, uint32_t n,
                                                 uint32_t vocab, float c, float* q, bool* some) {
    const uint32_t lane = threadIdx.x & 63;
    float v[kMaxSlots / 64], hi = -kInf;
#pragma unroll
    for (uint32_t r = 0; r < kMaxSlots / 64; ++r) {
        const uint32_t i = lane + 64 * r;
        v[r] = -kInf;
        if (i < n) {
            const int32_t id = ids[first + i];
            if (id >= 0 && (uint32_t)id < vocab) v[r] = teacher_logit(z, as_bf16, first + i);
        }
        hi = fmaxf(hi, v[r]);
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) hi = fmaxf(hi, __shfl_xor(hi, d));
    float sum = 0.f;
#pragma unroll
    for (uint32_t r = 0; r < kMaxSlots / 64; ++r)
        if (lane + 64 * r < n && v[r] != -kInf) sum += exp2_fast((v[r] - hi) * c);
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d);
    const float l = log2f(sum);
    float minus_entropy = 0.f;
#pragma unroll
    for (uint32_t r = 0; r < kMaxSlots / 64; ++r) {
        const uint32_t i = lane + 64 * r;
        if (i < n) {
            float qi = 0.f;
            if (v[r] != -kInf) {
                const float lq = (v[r] - hi) * c - l;
                qi = exp2_fast(lq);
                minus_entropy += qi * fmaxf(lq, -256.f);
            }
            q[i] = qi;
        }
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) minus_entropy += __shfl_xor(minus_entropy, d);
    *some = !(sum == 0.f);
    return minus_entropy;
}

struct RowGrad {
    float m, l, c;
    float whole;         // -s C
    float ent, H;        // -s g, entropy
    template <bool ENTROPY> __device__ __forceinline__ float at(float x) const {
        const float t = (x - m) * c - l, pr = exp2_fast(t);
        float d = whole * pr;
        if (ENTROPY) d = fmaf(ent * pr, fmaf(fmaxf(t, -256.f), kLn2, H), d);
        return d;
    }
};

// Writes vectors [v0, v1) (and the edge elements if `edges`) of a row's gradient, then the entries that tokens name.
// Same tokens add up in slot order, and the first of them writes the entry.  d may be x itself: the named logits are
// read before anything is written.
template <typename T, int THREADS, bool ENTROPY>
__device__ __forceinline__ void write_gradient(const RowSpan<T>& span, T* d, uint32_t v0, uint32_t v1, bool edges, bool zero,
                                               const RowGrad& g, const int32_t* ids, const float* coef, uint32_t n,
                                               uint32_t vocab, float s) {
    constexpr int N = LogitVec<T>::N;
    const uint32_t t = threadIdx.x;
    const int32_t edge = edges ? span.edge(t) : -1;
    if (zero) {   // nothing reaches this row (padding): its logits, whatever they hold, are not read
        for (uint32_t v = v0 + t; v < v1; v += THREADS) *(u32x4*)(d + span.index(v)) = u32x4{0, 0, 0, 0};
        if (edge >= 0) LogitVec<T>::store(d + edge, 0.f);
        return;
    }
    constexpr uint32_t ROUNDS = kMaxSlots / THREADS > 0 ? kMaxSlots / THREADS : 1;
    float named[ROUNDS];
    bool writes[ROUNDS];
    const uint32_t first = span.index(v0), last = span.index(v1);
#pragma unroll
    for (uint32_t r = 0; r < ROUNDS; ++r) {
        const uint32_t i = t + r * THREADS;
        writes[r] = false;
        if (i < n) {
            const int32_t id = ids[i];
            writes[r] = id >= 0 && (uint32_t)id < vocab &&
                        (((uint32_t)id >= first && (uint32_t)id < last) ||
                         (edges && ((uint32_t)id < span.head || (uint32_t)id >= span.index(span.vecs))));
            if (writes[r]) {
                float total = 0.f;
                for (uint32_t k = 0; k < n; ++k)
                    if (ids[k] == id) {
                        if (k < i) { writes[r] = false; break; }
                        total += coef[k];
                    }
                if (writes[r]) named[r] = fmaf(s, total, g.template at<ENTROPY>(LogitVec<T>::load(span.row + id)));
            }
        }
    }
    __syncthreads();
    for (uint32_t v = v0 + t; v < v1; v += THREADS) {
        float x[N];
        LogitVec<T>::unpack(span.vec(v), x);
#pragma unroll
        for (int u = 0; u < N; ++u) x[u] = g.template at<ENTROPY>(x[u]);
        *(u32x4*)(d + span.index(v)) = LogitVec<T>::pack(x);
    }
    if (edge >= 0) LogitVec<T>::store(d + edge, g.template at<ENTROPY>(LogitVec<T>::load(span.row + edge)));
    __syncthreads();
#pragma unroll
    for (uint32_t r = 0; r < ROUNDS; ++r)
        if (writes[r]) LogitVec<T>::store(d + ids[t + r * THREADS], named[r]);
}

template <typename T, int THREADS, bool ENTROPY, bool TEACHER>
__global__ __launch_bounds__(THREADS) void logit_gradient_kernel(GradParams p) {
    __shared__ float red[16];
    __shared__ float coef[kMaxSlots];
    __shared__ int32_t ids[kMaxSlots];
    const uint32_t t = threadIdx.x;
    const size_t row = blockIdx.x / p.chunks;
    const uint32_t chunk = blockIdx.x % p.chunks;
    const RowSpan<T> span((const T*)p.logits + row * p.stride, p.vocab);
    const uint32_t v0 = chunk * p.chunk_vecs < span.vecs ? chunk * p.chunk_vecs : span.vecs;
    const uint32_t v1 = v0 + p.chunk_vecs < span.vecs ? v0 + p.chunk_vecs : span.vecs;
    const float l = p.stats[2 * row + 1];
    RowGrad g;
    g.m = p.stats[2 * row];
    g.l = l;
    g.c = p.c;
    g.ent = ENTROPY ? -p.scale * p.d_entropy[row] : 0.f;
    g.H = ENTROPY ? p.entropy[row] : 0.f;
    float C = 0.f, any = 0.f;
    const float w = TEACHER ? p.d_loss[row] / (p.scale * p.scale) : 0.f;
    if (TEACHER) {
        if (t < 64) {
            bool some;
            teacher_softmax(p.ids, p.teacher, p.teacher_bf16, row * p.n, p.n, p.vocab, p.c, coef, &some);
            if (t == 0) red[0] = some ? 1.f : 0.f;
        }
        __syncthreads();
        if (red[0] != 0.f && w != 0.f) { C = -w; any = 1.f; }
        __syncthreads();
    }
    for (uint32_t i = t; i < p.n; i += THREADS) {
        const int32_t id = p.ids[row * p.n + i];
        ids[i] = id;
        if (TEACHER) {
            coef[i] *= -w;
        } else {
            const float v = id >= 0 && (uint32_t)id < p.vocab ? p.d_logprob[row * p.n + i] : 0.f;
            coef[i] = v;
            C += v;
            if (v != 0.f) any = 1.f;
        }
    }
    if (!TEACHER) {
        C = group_sum<THREADS>(C, red);
        any = group_max<THREADS>(any, red);
        if (g.ent != 0.f) any = 1.f;
    }
    __syncthreads();
    g.whole = -p.scale * C;
    write_gradient<T, THREADS, ENTROPY>(span, (T*)p.d_logits + row * p.stride, v0, v1, chunk == 0,
                                        any == 0.f || l == -kInf, g, ids, coef, p.n, p.vocab, p.scale);
}

// ---- distillation ---------------------------------------------------------------------------------------------
struct DistillParams {
    const void* logits;
    void* d_logits;          // or NULL
    const int32_t* ids;
    const void* teacher;
    const float* d_loss;
    float *row_loss, *stats;
    uint64_t stride;
    uint32_t vocab, n;
    int teacher_bf16;
    float scale, c;
};

// One work-group per row: the student's softmax sum, the loss over the teacher's slots, and (GRAD) the gradient in a
// second sweep over the row.
template <typename T, int THREADS, bool GRAD>
__global__ __launch_bounds__(THREADS) void distill_kernel(DistillParams p) {
    __shared__ float red[16];
    __shared__ float q[kMaxSlots];
    __shared__ int32_t ids[kMaxSlots];
    __shared__ uint32_t has_teacher;
    const uint32_t t = threadIdx.x;
    const size_t row = blockIdx.x;
    const RowSpan<T> span((const T*)p.logits + row * p.stride, p.vocab);
    float valid = 0.f;
    for (uint32_t i = t; i < p.n; i += THREADS) {
        const int32_t id = p.ids[row * p.n + i];
        ids[i] = id;
        if (id >= 0 && (uint32_t)id < p.vocab) valid = 1.f;
    }
    valid = group_max<THREADS>(valid, red);
    RowGrad g;
    g.m = g.l = -kInf;
    g.c = p.c;
    g.ent = g.H = 0.f;
    bool some = false;
    if (valid != 0.f) {   // (a row without a slot is padding: its logits are not read)
        const RowSum acc = sum_row<T, THREADS, false>(span, span.edge(t), p.c, red);
        g.m = acc.ref;
        g.l = log2f(acc.sum);
        float loss = 0.f;
        if (t < 64) {
            loss = teacher_softmax(p.ids, p.teacher, p.teacher_bf16, row * p.n, p.n, p.vocab, p.c, q, &some);
            float cross = 0.f;
            for (uint32_t i = t; i < p.n; i += 64)
                if (q[i] > 0.f || q[i] != q[i]) cross += q[i] * log_prob(LogitVec<T>::load(span.row + ids[i]), g.m, g.l, p.scale);
#pragma unroll
            for (int d = 32; d >= 1; d >>= 1) cross += __shfl_xor(cross, d);
            loss = some ? (loss * kLn2 - cross) / (p.scale * p.scale) : 0.f;
            if (t == 0) {
                p.row_loss[row] = loss;
                has_teacher = some ? 1u : 0u;
            }
        }
        __syncthreads();
        some = has_teacher != 0u;
    } else if (t == 0) {
        p.row_loss[row] = 0.f;
    }
    if (t == 0 && p.stats) { p.stats[2 * row] = g.m; p.stats[2 * row + 1] = g.l; }
    if (GRAD) {
        const float w = p.d_loss[row] / (p.scale * p.scale);
        for (uint32_t i = t; i < p.n; i += THREADS) q[i] *= -w;
        __syncthreads();
        g.whole = p.scale * w;
        write_gradient<T, THREADS, false>(span, (T*)p.d_logits + row * p.stride, 0, span.vecs, true,
                                          !some || w == 0.f || g.l == -kInf, g, ids, q, p.n, p.vocab, p.scale);
    }
}

// Threads of a row's work-group: a wave where a row is a few vectors per lane, more waves the longer it is.
static inline int row_threads(uint32_t vocab, int dtype) {
    const uint32_t vecs = vocab / (dtype == SFB_BF16 ? 8u : 4u);
    return vecs <= 512 ? 64 : vecs <= 16384 ? 256 : 1024;
}

static inline int check_logits(const void* logits, int dtype, uint64_t rows, uint32_t vocab, uint64_t stride, float scale,
                               const void* workspace = nullptr, size_t workspace_bytes = 0) {
    if (!logits) return SFB_ERR_NULL_POINTER;
    if (dtype != SFB_F32 && dtype != SFB_BF16) return SFB_ERR_DTYPE;
    if (rows == 0 || rows > 0x7fffffffull || vocab == 0 || vocab > 0x7fffffffu || stride < vocab) return SFB_ERR_SHAPE;
    if (stride > (1ull << 40)) return SFB_ERR_SHAPE;
    if (!(scale >= SFB_LOGIT_SCALE_MIN && scale <= SFB_LOGIT_SCALE_MAX)) return SFB_ERR_ARGUMENT;
    if (((uintptr_t)logits | (uintptr_t)workspace) & 15u) return SFB_ERR_ALIGNMENT;
    if (workspace && workspace_bytes < SFB_LOGIT_WORKSPACE_BYTES) return SFB_ERR_WORKSPACE;
    return SFB_OK;
}
static inline bool misaligned4(const void* a, const void* b = nullptr, const void* c = nullptr, const void* d = nullptr) {
    return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c | (uintptr_t)d) & 3u) != 0;
}

}  // namespace sfb

using namespace sfb;

#define SFB_ROW_THREADS(CALL)                                          \
    switch (row_threads(vocab, dtype)) {                               \
    case 64: CALL(64); break;                                          \
    case 256: CALL(256); break;                                        \
    default: CALL(1024); break;                                        \
    }

extern "C" int sfb_token_logprobs(sfb_stream_t stream, float* logprob, float* entropy, float* stats, int32_t* top_ids,
                                  float* top_logprobs, const void* logits, int dtype, const int32_t* tokens, uint64_t rows,
                                  uint32_t vocab, uint64_t row_stride, uint32_t n_tokens, uint32_t top_k, float scale,
                                  void* workspace, size_t workspace_bytes) {
    const int bad = check_logits(logits, dtype, rows, vocab, row_stride, scale, workspace, workspace_bytes);
    if (bad) return bad;
    if (n_tokens > kMaxSlots || top_k > kMaxTop || top_k > vocab) return SFB_ERR_SHAPE;
    if (n_tokens && (!logprob || !tokens)) return SFB_ERR_NULL_POINTER;
    if (top_k && (!top_ids || !top_logprobs)) return SFB_ERR_NULL_POINTER;
    if (!n_tokens && !top_k && !entropy && !stats) return SFB_ERR_ARGUMENT;
    if (misaligned4(logprob, entropy, stats, top_ids) || misaligned4(top_logprobs, tokens)) return SFB_ERR_ALIGNMENT;
    LogprobParams p{logits, tokens, logprob, entropy, stats, top_logprobs, top_ids, row_stride, vocab, n_tokens, top_k, scale,
                    scale * kLog2e};
    hipStream_t s = (hipStream_t)stream;
    clear_stale_error();
#define SFB_LP(TH)                                                                                          \
    do {                                                                                                    \
        if (dtype == SFB_F32) {                                                                             \
            if (entropy) token_logprobs_kernel<float, TH, true><<<dim3((uint32_t)rows), TH, 0, s>>>(p);     \
            else token_logprobs_kernel<float, TH, false><<<dim3((uint32_t)rows), TH, 0, s>>>(p);            \
        } else {                                                                                            \
            if (entropy) token_logprobs_kernel<__bf16, TH, true><<<dim3((uint32_t)rows), TH, 0, s>>>(p);    \
            else token_logprobs_kernel<__bf16, TH, false><<<dim3((uint32_t)rows), TH, 0, s>>>(p);           \
        }                                                                                                   \
    } while (0)
    SFB_ROW_THREADS(SFB_LP)
#undef SFB_LP
    return launch_status();
}

// Vectors of a row that one work-group of the backward pass writes.
static inline uint32_t grad_chunk_vecs(uint32_t) { return 1024; }

static int launch_gradient(hipStream_t s, GradParams& p, int dtype, uint64_t rows, bool entropy, bool teacher) {
    const uint32_t per = dtype == SFB_BF16 ? 8 : 4;
    p.chunk_vecs = grad_chunk_vecs(p.vocab);
    p.chunks = (p.vocab / per + p.chunk_vecs - 1) / p.chunk_vecs;
    if (p.chunks == 0) p.chunks = 1;
    if (rows * p.chunks > 0x7fffffffull) return SFB_ERR_SHAPE;
    const dim3 grid((uint32_t)(rows * p.chunks));
    clear_stale_error();
    if (dtype == SFB_F32) {
        if (teacher) logit_gradient_kernel<float, 256, false, true><<<grid, 256, 0, s>>>(p);
        else if (entropy) logit_gradient_kernel<float, 256, true, false><<<grid, 256, 0, s>>>(p);
        else logit_gradient_kernel<float, 256, false, false><<<grid, 256, 0, s>>>(p);
    } else {
        if (teacher) logit_gradient_kernel<__bf16, 256, false, true><<<grid, 256, 0, s>>>(p);
        else if (entropy) logit_gradient_kernel<__bf16, 256, true, false><<<grid, 256, 0, s>>>(p);
        else logit_gradient_kernel<__bf16, 256, false, false><<<grid, 256, 0, s>>>(p);
    }
    return launch_status();
}

extern "C" int sfb_token_logprobs_backward(sfb_stream_t stream, void* d_logits, const void* logits, int dtype,
                                           const int32_t* tokens, const float* stats, const float* entropy,
                                           const float* d_logprob, const float* d_entropy, uint64_t rows, uint32_t vocab,
                                           uint64_t row_stride, uint32_t n_tokens, float scale) {
    const int bad = check_logits(logits, dtype, rows, vocab, row_stride, scale);
    if (bad) return bad;
    if (!d_logits || !stats) return SFB_ERR_NULL_POINTER;
    if (n_tokens > kMaxSlots) return SFB_ERR_SHAPE;
    if (n_tokens && (!tokens || !d_logprob)) return SFB_ERR_NULL_POINTER;
    if (d_entropy && !entropy) return SFB_ERR_NULL_POINTER;
    if (!n_tokens && !d_entropy) return SFB_ERR_ARGUMENT;
    if ((uintptr_t)d_logits & 15u || misaligned4(tokens, stats, entropy, d_logprob) || misaligned4(d_entropy)) return SFB_ERR_ALIGNMENT;
    GradParams p{};
    p.logits = logits; p.d_logits = d_logits; p.ids = tokens; p.stats = stats; p.entropy = entropy; p.d_entropy = d_entropy;
    p.d_logprob = d_logprob; p.stride = row_stride; p.vocab = vocab; p.n = n_tokens; p.scale = scale; p.c = scale * kLog2e;
    return launch_gradient((hipStream_t)stream, p, dtype, rows, d_entropy != nullptr, false);
}

extern "C" int sfb_distillation_loss(sfb_stream_t stream, float* row_loss, float* stats, void* d_logits, const void* logits,
                                     int dtype, const int32_t* teacher_ids, const void* teacher_logits, int teacher_dtype,
                                     const float* d_loss, uint64_t rows, uint32_t vocab, uint64_t row_stride,
                                     uint32_t slots, float scale, void* workspace, size_t workspace_bytes) {
    const int bad = check_logits(logits, dtype, rows, vocab, row_stride, scale, workspace, workspace_bytes);
    if (bad) return bad;
    if (teacher_dtype != SFB_F32 && teacher_dtype != SFB_BF16) return SFB_ERR_DTYPE;
    if (slots == 0 || slots > kMaxSlots) return SFB_ERR_SHAPE;
    if (!row_loss || !teacher_ids || !teacher_logits || (d_logits && !d_loss)) return SFB_ERR_NULL_POINTER;
    if ((uintptr_t)d_logits & 15u || misaligned4(row_loss, stats, teacher_ids, d_loss) ||
        ((uintptr_t)teacher_logits & (teacher_dtype == SFB_BF16 ? 1u : 3u)))
        return SFB_ERR_ALIGNMENT;
    DistillParams p{logits, d_logits, teacher_ids, teacher_logits, d_loss, row_loss, stats, row_stride, vocab, slots,
                    teacher_dtype == SFB_BF16 ? 1 : 0, scale, scale * kLog2e};
    hipStream_t s = (hipStream_t)stream;
    clear_stale_error();
#define SFB_DL(TH)                                                                                     \
    do {                                                                                               \
        if (dtype == SFB_F32) {                                                                        \
            if (d_logits) distill_kernel<float, TH, true><<<dim3((uint32_t)rows), TH, 0, s>>>(p);      \
            else distill_kernel<float, TH, false><<<dim3((uint32_t)rows), TH, 0, s>>>(p);              \
        } else {                                                                                       \
            if (d_logits) distill_kernel<__bf16, TH, true><<<dim3((uint32_t)rows), TH, 0, s>>>(p);     \
            else distill_kernel<__bf16, TH, false><<<dim3((uint32_t)rows), TH, 0, s>>>(p);             \
        }                                                                                              \
    } while (0)
    SFB_ROW_THREADS(SFB_DL)
#undef SFB_DL
    return launch_status();
}

extern "C" int sfb_distillation_loss_backward(sfb_stream_t stream, void* d_logits, const void* logits, int dtype,
                                              const int32_t* teacher_ids, const void* teacher_logits, int teacher_dtype,
                                              const float* stats, const float* d_loss, uint64_t rows, uint32_t vocab,
                                              uint64_t row_stride, uint32_t slots, float scale) {
    const int bad = check_logits(logits, dtype, rows, vocab, row_stride, scale);
    if (bad) return bad;
    if (teacher_dtype != SFB_F32 && teacher_dtype != SFB_BF16) return SFB_ERR_DTYPE;
    if (slots == 0 || slots > kMaxSlots) return SFB_ERR_SHAPE;
    if (!d_logits || !stats || !d_loss || !teacher_ids || !teacher_logits) return SFB_ERR_NULL_POINTER;
    if ((uintptr_t)d_logits & 15u || misaligned4(stats, d_loss, teacher_ids) ||
        ((uintptr_t)teacher_logits & (teacher_dtype == SFB_BF16 ? 1u : 3u)))
        return SFB_ERR_ALIGNMENT;
    GradParams p{};
    p.logits = logits; p.d_logits = d_logits; p.ids = teacher_ids; p.stats = stats; p.teacher = teacher_logits;
    p.teacher_bf16 = teacher_dtype == SFB_BF16 ? 1 : 0; p.d_loss = d_loss; p.stride = row_stride; p.vocab = vocab;
    p.n = slots; p.scale = scale; p.c = scale * kLog2e;
    return launch_gradient((hipStream_t)stream, p, dtype, rows, false, true);
}
