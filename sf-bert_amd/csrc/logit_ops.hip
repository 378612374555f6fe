// Operators on rows of logits: the log probabilities of given tokens with entropy and top alternatives, and the
// distillation loss against a teacher's top logits, each with its gradient.  No counterpart in the reference, whose
// only loss is softmax_cross_entropy_with_logits (ewops.h:233-261).
//
// With s = scale, c = s log2(e), a row x and any reference m:  S = sum_j 2^((x_j - m) c),  l = log2 S,
//   ln p_j = (x_j - m) s - ln2 l,   entropy = ln2 (l - W / S) with W = sum_j 2^t_j t_j, t_j = (x_j - m) c.
// Everything is held in fp32.  The row is read once; (m, l) is what the backward pass is given.
//
// What bounds these kernels is reading the rows (and writing gradients): this card reads 7.1 TB/s and copies 6.2 with
// nontemporal accesses, 6.3 and 5.6 with plain ones, so every row's vectors are loaded and stored nontemporally.
#include "common.hip.h"

namespace sfb {

constexpr uint32_t kMaxTop = 64;      // alternatives per row
constexpr uint32_t kMaxSlots = 256;   // given tokens, or entries of a teacher's list, per row
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kInf = __builtin_inff();
// A reference's scaled value m c is rounded, and what rounding leaves out must stay a small exponent: up to kWide that is
// at most one.  Rows whose largest scaled logit passes kWide in either direction are left to a second pass that subtracts
// the maximum before it scales.  kNoReference: the scaled reference of a lane that has not met a logit above it yet; in
// all other rows what stays below it is at least kWide powers of two from the largest logit.
constexpr float kWide = 0x1p24f;
constexpr float kNoReference = -0x1p25f;

// A 16-byte vector of logits.
template <typename T> struct LogitVec;
template <> struct LogitVec<float> {
    static constexpr int N = 4;
    static constexpr uint32_t kMasked = 0xff800000u;   // -inf
    static constexpr uint32_t kMaskedOne = kMasked;
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
    // one logit's bits and their value (apart, so that a load need not be waited for where it is issued)
    __device__ static __forceinline__ uint32_t bits(const float* p) { return *(const uint32_t*)p; }
    __device__ static __forceinline__ float value(uint32_t b) { return __builtin_bit_cast(float, b); }
    __device__ static __forceinline__ float load(const float* p) { return *p; }
    __device__ static __forceinline__ void store(float* p, float v) { *p = v; }
};
template <> struct LogitVec<__bf16> {
    static constexpr int N = 8;
    static constexpr uint32_t kMasked = 0xff80ff80u;   // -inf, twice
    static constexpr uint32_t kMaskedOne = 0xff80u;
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
    __device__ static __forceinline__ uint32_t bits(const __bf16* p) { return *(const uint16_t*)p; }
    __device__ static __forceinline__ float value(uint32_t b) { return bf16_bits_to_f32(b); }
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
    // the same division of another row with the same alignment
    __device__ __forceinline__ RowSpan onto(const T* r) const {
        RowSpan s(*this);
        s.row = r;
        return s;
    }
    // element index of the edge element thread t takes care of (one each), or -1
    __device__ __forceinline__ int32_t edge(uint32_t t) const {
        if (t < head) return (int32_t)t;
        if (t < head + tail) return (int32_t)(head + vecs * LogitVec<T>::N + (t - head));
        return -1;
    }
    // vector `base + i`, base the same for the whole wave: its address stays in scalar registers
    __device__ __forceinline__ const u32x4* at(uint32_t base, uint32_t i) const {
        return (const u32x4*)((const char*)(row + head) + (size_t)base * 16 + i * 16);
    }
    __device__ __forceinline__ uint32_t index(uint32_t i) const { return head + i * LogitVec<T>::N; }
};

// The part of a row one work-group takes: vectors [v0, v1) and elements [e0, e1), which add the row's first elements to
// the first part and its last ones to the last.
struct Slice {
    uint32_t v0, v1, e0, e1;
    int32_t edge;   // the edge element of this thread, or -1
};
template <typename T>
__device__ __forceinline__ Slice slice_of(const RowSpan<T>& span, uint32_t vocab, uint32_t part, uint32_t parts, uint32_t each,
                                          uint32_t t) {
    Slice s;
    s.v0 = part * each < span.vecs ? part * each : span.vecs;
    s.v1 = part + 1 == parts || s.v0 + each > span.vecs ? span.vecs : s.v0 + each;
    s.e0 = part == 0 ? 0 : span.index(s.v0);
    s.e1 = part + 1 == parts ? vocab : span.index(s.v1);
    s.edge = span.edge(t);
    if (s.edge >= 0 && ((uint32_t)s.edge < s.e0 || (uint32_t)s.edge >= s.e1)) s.edge = -1;
    return s;
}

// ---- reductions -----------------------------------------------------------------------------------------------
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane(float v, int i) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), i));
}
// Within 16 lanes by DPP moves (neighbours, pairs, mirrored halves), the four results by lane reads: no LDS round trips.
// All lanes get the same bits.
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, dpp<0xB1>(v));
    v = fmaxf(v, dpp<0x4E>(v));
    v = fmaxf(v, dpp<0x141>(v));
    v = fmaxf(v, dpp<0x140>(v));
    return fmaxf(fmaxf(lane(v, 0), lane(v, 16)), fmaxf(lane(v, 32), lane(v, 48)));
}
__device__ __forceinline__ float wave_sum(float v) {
    v += dpp<0xB1>(v);
    v += dpp<0x4E>(v);
    v += dpp<0x141>(v);
    v += dpp<0x140>(v);
    return (lane(v, 0) + lane(v, 16)) + (lane(v, 32) + lane(v, 48));
}
// red: THREADS / 64 floats for max, twice that for sums.  Sums are taken in an order that depends on THREADS alone.
// publish() is called between the two barriers, by every thread.
template <int THREADS, typename P> __device__ __forceinline__ float group_max(float v, float* red, P publish) {
    v = wave_max(v);
    __syncthreads();
    if (THREADS > 64 && (threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    publish();
    __syncthreads();
    if (THREADS == 64) return v;
    v = red[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) v = fmaxf(v, red[w]);
    return v;
}
template <int THREADS, bool BOTH> __device__ __forceinline__ void group_sum(float& a, float& b, float* red) {
    a = wave_sum(a);
    if (BOTH) b = wave_sum(b);
    if (THREADS == 64) return;
    constexpr int W = THREADS / 64;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        red[threadIdx.x >> 6] = a;
        if (BOTH) red[W + (threadIdx.x >> 6)] = b;
    }
    __syncthreads();
    a = red[0];
    if (BOTH) b = red[W];
#pragma unroll
    for (int w = 1; w < W; ++w) {
        a += red[w];
        if (BOTH) b += red[W + w];
    }
}

// ---- the softmax sums of a row --------------------------------------------------------------------------------
struct RowSum {
    float m;           // reference logit (-inf: nothing but -inf and NaN)
    float sum, dot;    // sum 2^t, sum 2^t t with t = (x - m) c
    float top;         // this thread's largest logit (NaN left out)
};

template <int N> __device__ __forceinline__ float largest(const float (&x)[N]) {
    float hi = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) hi = fmaxf(hi, x[i]);
    return hi;
}
template <typename T, int G> __device__ __forceinline__ float largest_of(const u32x4* raw) {
    float hi = -kInf;
#pragma unroll
    for (int u = 0; u < G; ++u) {
        float x[LogitVec<T>::N];
        LogitVec<T>::unpack(raw[u], x);
        hi = fmaxf(hi, largest(x));
    }
    return hi;
}

// 2^t and 2^t t; t = -inf (a masked logit) stands for 0 in both, a NaN reaches both.
template <bool ENTROPY, bool CLAMP = true> __device__ __forceinline__ void add_term(float t, float& sum, float& dot) {
    const float e = exp2_fast(t);
    sum += e;
    if (ENTROPY) dot = fmaf(e, CLAMP ? fmaxf(t, -256.f) : t, dot);
}
// The terms of G vectors relative to ref2.  Clamping t costs a seventh of the entropy's instructions and is for masked
// logits alone, so it is left out until a 0 * -inf shows that there are some: that step is then done again, and the
// wave clamps from there on.
template <typename T, int G, bool ENTROPY>
__device__ __forceinline__ void add_terms(const u32x4* raw, float c, float ref2, float& sum, float& dot, bool& clamp) {
    constexpr int N = LogitVec<T>::N;
    const float sum0 = sum, dot0 = dot;
    if (!ENTROPY || !clamp) {
#pragma unroll
        for (int u = 0; u < G; ++u) {
            float x[N];
            LogitVec<T>::unpack(raw[u], x);
#pragma unroll
            for (int i = 0; i < N; ++i) add_term<ENTROPY, false>(fmaf(x[i], c, -ref2), sum, dot);
        }
        if (!ENTROPY || __builtin_amdgcn_ballot_w64(dot != dot) == 0) return;
        clamp = true;
        sum = sum0;
        dot = dot0;
    }
#pragma unroll
    for (int u = 0; u < G; ++u) {
        u32x4 again = raw[u];
        asm volatile("" : "+v"(again));   // (nothing of the first attempt is kept in registers for this one)
        float x[N];
        LogitVec<T>::unpack(again, x);
#pragma unroll
        for (int i = 0; i < N; ++i) add_term<ENTROPY, true>(fmaf(x[i], c, -ref2), sum, dot);
    }
}

// Rows whose logits are subtracted from the maximum before they are scaled.
__device__ __forceinline__ bool is_wide(float m, float c) { return fabsf(m * c) > kWide && fabsf(m) < kInf; }

template <int V> struct Int { static constexpr int value = V; };

// G vectors of every thread, `base` the first thread's first vector, THREADS apart.  The loads are unconditional (past
// the end: the last vector), so that all of them are in flight at once.  Logits are read once: nontemporal loads.
template <typename T, int THREADS, int G>
__device__ __forceinline__ void load_vectors(const RowSpan<T>& span, const Slice& s, uint32_t base, uint32_t t, u32x4* raw) {
#pragma unroll
    for (int u = 0; u < G; ++u) {
        const uint32_t b = base + u * THREADS < s.v1 ? base + u * THREADS : s.v1 - 1, last = s.v1 - 1 - b;
        raw[u] = __builtin_nontemporal_load(span.at(b, t < last ? t : last));
    }
}
// f(count, vectors, base) for these G vectors: all at once where the work-group has all of them, else one by one as far
// as the slice goes.  MASK: what lies past its end is first overwritten with -inf, which counts nowhere.
template <typename T, int THREADS, int G, bool MASK, typename F>
__device__ __forceinline__ void step_vectors(const Slice& s, uint32_t base, uint32_t t, u32x4* raw, F f) {
    if (base + G * THREADS <= s.v1) {
        f(Int<G>(), raw, base);
        return;
    }
#pragma unroll
    for (int u = 0; u < G; ++u) {
        const uint32_t b = base + u * THREADS;
        if (b < s.v1) {
            if (MASK && b + t >= s.v1) raw[u] = u32x4{LogitVec<T>::kMasked, LogitVec<T>::kMasked, LogitVec<T>::kMasked, LogitVec<T>::kMasked};
            f(Int<1>(), raw + u, b);
        }
    }
}

// A slice held in registers: NV vectors per thread, read before anything is computed, so that the maximum is known when
// the exponentials begin.
template <typename T, int THREADS, int NV> struct Held {
    static constexpr int N = LogitVec<T>::N;
    static constexpr int G = NV < 2 ? NV : 2;   // vectors per step
    u32x4 raw[NV];
    uint32_t edge;   // bits of the edge element
    __device__ __forceinline__ void load(const RowSpan<T>& span, const Slice& s, uint32_t t) {
        edge = LogitVec<T>::kMaskedOne;
        if (s.edge >= 0) edge = LogitVec<T>::bits(span.row + s.edge);
        if (s.v1 > s.v0) load_vectors<T, THREADS, NV>(span, s, s.v0, t, raw);
    }
    // f(x, base, vector) for every vector of this thread, which is the t-th from base
    template <typename F> __device__ __forceinline__ void each(const Slice& s, uint32_t t, F f) const {
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const uint32_t base = s.v0 + u * THREADS;
            if (base + t < s.v1) {
                float x[N];
                LogitVec<T>::unpack(raw[u], x);
                f(x, base);
            }
        }
    }
    template <bool MASK, typename F> __device__ __forceinline__ void steps(const Slice& s, uint32_t t, F f) {
#pragma unroll
        for (int g = 0; g < NV; g += G)
            if (s.v0 + g * THREADS < s.v1) step_vectors<T, THREADS, G, MASK>(s, s.v0 + g * THREADS, t, raw + g, f);
    }
    // publish(largest logit) is called by every thread before the work-group meets for the maximum, met(maximum) right
    // after (what it leaves in shared memory can be read when the sums are there).  EXTRA: dot is the work-group's sum of
    // what met() returns.
    template <bool ENTROPY, bool EXTRA, typename P, typename M>
    __device__ __forceinline__ RowSum sums(const Slice& s, uint32_t t, float c, float* red, P publish, M met) {
        RowSum r;
        const float single = LogitVec<T>::value(edge);
        r.top = single;
        steps<true>(s, t, [&](auto count, const u32x4* x, uint32_t) { r.top = fmaxf(r.top, largest_of<T, decltype(count)::value>(x)); });
        r.m = group_max<THREADS>(r.top, red, [&]() { publish(r.top); });
        const float m = r.m == -kInf ? 0.f : r.m;
        const float extra = met(m);
        r.sum = r.dot = 0.f;
        if (!is_wide(m, c)) {
            const float mc = m * c, d = fmaf(m, c, -mc);   // d: what rounding left out of m c
            bool clamp = false;
            steps<false>(s, t, [&](auto count, const u32x4* x, uint32_t) {
                add_terms<T, decltype(count)::value, ENTROPY>(x, c, mc, r.sum, r.dot, clamp);
            });
            add_term<ENTROPY>(fmaf(single, c, -mc), r.sum, r.dot);
            const float f = exp2_fast(-d);
            if (ENTROPY) r.dot = f * (r.dot - d * r.sum);
            r.sum *= f;
        } else {
            each(s, t, [&](const float (&x)[N], uint32_t) {
#pragma unroll
                for (int i = 0; i < N; ++i) add_term<ENTROPY>((x[i] - m) * c, r.sum, r.dot);
            });
            add_term<ENTROPY>((single - m) * c, r.sum, r.dot);
        }
        if (EXTRA) r.dot = extra;
        group_sum<THREADS, ENTROPY || EXTRA>(r.sum, r.dot, red);
        return r;
    }
};

// A row longer than the registers of its work-group, in one pass.  Each thread keeps its sums relative to a reference of
// its own that lags its largest logit by at most kLazyRescaleLog2 powers of two, so that it hardly ever moves after the
// first step.
template <typename T, int THREADS> struct Streamed {
    static constexpr int N = LogitVec<T>::N;
    static constexpr int G = 4, P = 2;   // vectors in flight, and per step

    // f(x, base) for every vector of this thread, as above
    template <typename F> static __device__ __forceinline__ void each(const RowSpan<T>& span, const Slice& s, uint32_t t, F f) {
        for (uint32_t base = s.v0; base < s.v1; base += THREADS * G) {
            u32x4 raw[G];
            load_vectors<T, THREADS, G>(span, s, base, t, raw);
#pragma unroll
            for (int u = 0; u < G; ++u)
                if (base + u * THREADS + t < s.v1) {
                    float x[N];
                    LogitVec<T>::unpack(raw[u], x);
                    f(x, base + u * THREADS);
                }
        }
    }
    // early(f) is called once, by every thread, f() giving its largest logit among the first vectors; meet(count, vectors,
    // largest, base) for what every step holds.
    // EXTRA, met: as above.
    template <bool ENTROPY, bool EXTRA, typename E, typename M, typename F>
    static __device__ __forceinline__ RowSum sums(const RowSpan<T>& span, const Slice& s, uint32_t t, float c, float* red, E early, M meet,
                                                  F met) {
        RowSum r;
        r.top = -kInf;
        r.sum = r.dot = 0.f;
        float ref = -kInf, ref2 = kNoReference;   // the reference logit and fl(ref c)
        bool clamp = false;
        auto raise = [&](float hi) {
            r.top = fmaxf(r.top, hi);
            const float hi2 = hi * c;
            const bool higher = hi2 > ref2 + kLazyRescaleLog2;
            if (__builtin_amdgcn_ballot_w64(higher) != 0) {   // (a branch of the whole wave, hardly ever taken)
                asm volatile("" : : : "memory");   // (kept a branch: made a select, it would cost every step)
                if (higher) {
                    const float d = ref2 - hi2, f = exp2_fast(d);
                    if (ENTROPY) r.dot = f * (r.dot + fmaxf(d, -256.f) * r.sum);
                    r.sum *= f;
                    ref = hi;
                    ref2 = hi2;
                }
            }
        };
        uint32_t edge = LogitVec<T>::kMaskedOne;
        if (s.edge >= 0) edge = LogitVec<T>::bits(span.row + s.edge);
        auto step = [&](auto count, const u32x4* raw, uint32_t base) {
            const float hi = largest_of<T, decltype(count)::value>(raw);
            raise(hi);
            meet(count, raw, hi, base);
            add_terms<T, decltype(count)::value, ENTROPY>(raw, c, ref2, r.sum, r.dot, clamp);
        };
        auto steps = [&](u32x4* raw, uint32_t base) {
#pragma unroll
            for (int g = 0; g < G; g += P)
                if (base + g * THREADS < s.v1) step_vectors<T, THREADS, P, true>(s, base + g * THREADS, t, raw + g, step);
        };
        if (s.v1 > s.v0) {
            u32x4 raw[2 * G];
            load_vectors<T, THREADS, 2 * G>(span, s, s.v0, t, raw);
            early([&]() {
                float hi = LogitVec<T>::value(edge);
                auto top = [&](auto count, const u32x4* x, uint32_t) { hi = fmaxf(hi, largest_of<T, decltype(count)::value>(x)); };
                step_vectors<T, THREADS, G, true>(s, s.v0, t, raw, top);
                if (s.v0 + G * THREADS < s.v1) step_vectors<T, THREADS, G, true>(s, s.v0 + G * THREADS, t, raw + G, top);
                return hi;
            });
            steps(raw, s.v0);
            if (s.v0 + G * THREADS < s.v1) steps(raw + G, s.v0 + G * THREADS);
        } else {
            early([&]() { return LogitVec<T>::value(edge); });
        }
        for (uint32_t base = s.v0 + 2 * THREADS * G; base < s.v1; base += THREADS * G) {
            u32x4 raw[G];
            load_vectors<T, THREADS, G>(span, s, base, t, raw);
            steps(raw, base);
        }
        const float single = LogitVec<T>::value(edge);
        raise(single);
        add_term<ENTROPY>(fmaf(single, c, -ref2), r.sum, r.dot);
        const float top = group_max<THREADS>(r.top, red, []() {});
        if (is_wide(top, c)) {
            r.sum = r.dot = 0.f;
            each(span, s, t, [&](const float (&x)[N], uint32_t) {
#pragma unroll
                for (int i = 0; i < N; ++i) add_term<ENTROPY>((x[i] - top) * c, r.sum, r.dot);
            });
            if (s.edge >= 0) add_term<ENTROPY>((single - top) * c, r.sum, r.dot);
        } else if (ref != -kInf) {   // from the thread's fl(ref c) to the row's largest logit
            const float rounding = fmaf(ref, c, -ref2);
            const float d = ref == top ? -rounding : (ref - top) * c - rounding, f = exp2_fast(d);
            if (ENTROPY) r.dot = f * (r.dot + fmaxf(d, -256.f) * r.sum);
            r.sum *= f;
        } else {   // nothing near the row's largest logit: no share in the sums but a NaN's
            r.sum = r.dot = r.sum == r.sum ? 0.f : r.sum;
        }
        r.m = top;
        if (EXTRA) r.dot = met(top == -kInf ? 0.f : top);
        group_sum<THREADS, ENTROPY || EXTRA>(r.sum, r.dot, red);
        return r;
    }
};

// Order of the alternatives as whole numbers: larger logits first, -0 as +0, NaN above everything; 0 is below every
// logit.  A composite's low word is the complement of the index: of equal logits the lowest index comes first.
constexpr uint32_t kMaskedOrder = 0x007fffffu;   // of -inf
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
    if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t order) {
    return __builtin_bit_cast(float, order & 0x80000000u ? (order == 0xffffffffu ? 0x7fc00000u : order & 0x7fffffffu) : ~order);
}
__device__ __forceinline__ uint64_t composite(uint32_t order, uint32_t index) { return ((uint64_t)order << 32) | (uint32_t)~index; }

// The k largest of a slice whose threads know the largest logit each of them has met.  The largest logits of 64 or 256
// groups of threads are compared: the k-th largest of those is at most the slice's k-th largest logit, and hardly more
// than k logits reach it (256 groups and k = 20: 21 expected), so only the threads whose own largest does look at their
// vectors again.  A slice with more equal or clustered logits than the list holds takes the exact threshold instead.
// HELD: vectors per thread, where that is all there are (0: more).
template <typename T, int THREADS, int HELD> struct TopSelect {
    static constexpr int N = LogitVec<T>::N;
    // (shared memory bounds how many short rows a compute unit works on at a time)
    static constexpr int VECTORS = HELD && HELD * THREADS < 256 ? HELD * THREADS : 256;
    static constexpr int LIST = HELD && HELD * THREADS * N + 16 < 512 ? HELD * THREADS * N + 16 : 512;
    // (one or two waves that hold a row give several groups each thread: with 64 groups and 64 alternatives the
    // threshold is the least of the threads' maxima: 8000 rows of 2000 took 880 us, take 36)
    static constexpr int PER = HELD >= 4 && THREADS < 256 ? 256 / THREADS : 1;
    static constexpr int GROUPS = THREADS * PER < 256 ? THREADS * PER : 256;
    static constexpr uint32_t THIN = 128;
    static constexpr uint32_t kBetween = 0, kExact = 1, kCommon = 2;
    static constexpr int LOW_BIT = sizeof(T) == 2 ? 16 : 0;   // bf16 logits are told apart by the upper half
    static_assert(GROUPS <= VECTORS, "the groups share memory with the vectors");
    struct Shared {
        u32x4 vectors[VECTORS];       // vectors that hold a logit above the threshold
        uint64_t list[LIST];          // composites
        uint32_t at[VECTORS];         // index of each vector's first element; before: the groups' largest logits
        uint32_t limit, kind;         // the threshold
        uint32_t count, n_vectors;
    };
    static __device__ __forceinline__ Shared& shared() {
        __shared__ Shared memory;
        return memory;
    }

    static __device__ __forceinline__ void append(uint32_t order, uint32_t index) {
        const uint32_t at = __hip_atomic_fetch_add(&shared().count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        if (at < (uint32_t)LIST) shared().list[at] = composite(order, index);
    }
    static __device__ __forceinline__ void clear_count() {
        __syncthreads();
        if (threadIdx.x == 0) shared().count = 0;
        __syncthreads();
    }

    // The largest value that at least k of 64 * W groups' largest logits reach, found bit by bit by one wave; it ends
    // early where exactly k reach it (*kind = kBetween: the threshold need not be one of them).  kExact: it is one;
    // kCommon: it is that of half of the groups, which is what a mask leaves (or rows of few different values).
    template <int W> static __device__ __forceinline__ uint32_t search(uint32_t k, uint32_t* kind) {
        uint32_t own[W], limit = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) own[i] = shared().at[i * 64 + (threadIdx.x & 63)];
        *kind = kExact;
        for (int bit = 31; bit >= LOW_BIT; --bit) {
            const uint32_t next = limit | (1u << bit);
            uint32_t n = 0;
#pragma unroll
            for (int i = 0; i < W; ++i) n += (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(own[i] >= next));
            if (n >= k) limit = next;
            if (n == k) { *kind = kBetween; break; }
        }
        // (orders of negative bf16 logits end in ones)
        if (LOW_BIT && !(limit >> 31)) limit |= (1u << LOW_BIT) - 1;
        if (*kind == kExact && limit >= kMaskedOrder) {
            uint32_t n = 0, there = 0;
#pragma unroll
            for (int i = 0; i < W; ++i) {
                n += (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(own[i] == limit));
                there += (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(own[i] != 0));
            }
            if (2 * n >= there) *kind = kCommon;
        }
        return limit;
    }
    // A threshold that at least k logits of the threads' largest reach, in three parts with a barrier after the first and
    // the second: every thread publishes its largest logit (and count is cleared), one wave searches, all read the
    // result.  Up to k = 32 the threads form 64 groups (k = 20: 24 logits expected
    // above the threshold), beyond that up to 256; own(i): order of the i-th of this thread's PER groups.
    template <typename F> static __device__ __forceinline__ void publish(float top, bool any, uint32_t k, F own) {
        const uint32_t t = threadIdx.x;
        if (PER > 1 && k > 32) {
#pragma unroll
            for (int i = 0; i < PER; ++i) shared().at[i * THREADS + t] = own(i);
            if (t == 0) shared().count = shared().n_vectors = 0;
            return;
        }
        uint32_t mine = any ? order_of(top) : 0u;
        const bool wide = THREADS > 64 && k > 32;   // (THREADS >= 256)
        if (THREADS >= 128) mine = pair_max<0xB1>(mine, THREADS >= 512 || !wide);
        if (THREADS >= 256) mine = pair_max<0x4E>(mine, THREADS >= 1024 || !wide);
        if (THREADS >= 512 && !wide) mine = pair_max<0x141>(mine, true);
        if (THREADS >= 1024 && !wide) mine = pair_max<0x140>(mine, true);
        const uint32_t per = wide ? THREADS / GROUPS : THREADS / 64;
        if (t % per == 0) shared().at[t / per] = mine;
        if (t == 0) shared().count = shared().n_vectors = 0;
    }
    static __device__ __forceinline__ void find(uint32_t k) {
        if (threadIdx.x >= 64) return;
        uint32_t kind;
        const uint32_t limit = GROUPS > 64 && k > 32 ? search<GROUPS / 64>(k, &kind) : search<1>(k, &kind);
        if (threadIdx.x == 0) { shared().limit = limit; shared().kind = kind; }
    }
    static __device__ __forceinline__ uint32_t found(uint32_t* kind) {
        *kind = shared().kind;
        return shared().limit;
    }
    static __device__ __forceinline__ uint32_t threshold(float top, bool any, uint32_t k, uint32_t* kind) {
        __syncthreads();
        publish(top, any, k, [](int) { return 0u; });
        __syncthreads();
        find(k);
        __syncthreads();
        return found(kind);
    }
    template <int CTRL> static __device__ __forceinline__ uint32_t pair_max(uint32_t v, bool take) {
        const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
        return take && o > v ? o : v;
    }

    // appends the logits of one vector that reach `least`
    static __device__ __forceinline__ void scan(const float (&x)[N], uint32_t index, float least) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (x[i] >= least) append(order_of(x[i]), index + i);
    }

    // What follows reads the slice again, element by element in groups of consecutive ones.
    template <typename F> static __device__ __forceinline__ void elements(const RowSpan<T>& span, const Slice& s, F f) {
        for (uint32_t j0 = s.e0; j0 < s.e1; j0 += THREADS) {
            const uint32_t j = j0 + threadIdx.x;
            if (!f(j < s.e1 ? order_of(LogitVec<T>::load(span.row + j)) : 0u, j)) break;
        }
    }
    static __device__ uint32_t reaching(const RowSpan<T>& span, const Slice& s, uint32_t limit) {
        uint32_t n = 0;
        elements(span, s, [&](uint32_t order, uint32_t) { n += order >= limit; return true; });
        clear_count();
        if (n) __hip_atomic_fetch_add(&shared().count, n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        __syncthreads();
        return shared().count;
    }
    // The k-th largest value, of which it is known that `from` is not above it, digit by digit from the highest: how many
    // values share the digits so far and have which next one.
    static __device__ uint32_t kth_largest(const RowSpan<T>& span, const Slice& s, uint32_t k, uint32_t from) {
        constexpr int BITS = VECTORS >= 256 ? 8 : 6;
        constexpr uint32_t BINS = 1u << BITS, SHARE = BINS / 16;
        static_assert(BINS <= VECTORS, "the counts share memory with the vectors");
        const uint32_t t = threadIdx.x;
        uint32_t value = 0, left = k;
        for (int high = 32; high > 0;) {
            const int low = high > BITS ? high - BITS : 0;
            const uint32_t known = high == 32 ? 0u : ~0u << high, digits = (1u << (high - low)) - 1;
            __syncthreads();
            for (uint32_t i = t; i < BINS; i += THREADS) shared().at[i] = 0;
            __syncthreads();
            elements(span, s, [&](uint32_t order, uint32_t j) {
                if (j < s.e1 && order >= from && ((order ^ value) & known) == 0)
                    __hip_atomic_fetch_add(&shared().at[order >> low & digits], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                return true;
            });
            __syncthreads();
            if (t < 16) {   // (the list is free: what it held was too much)
                uint32_t sum = 0;
                for (uint32_t i = 0; i < SHARE; ++i) sum += shared().at[t * SHARE + i];
                shared().list[t] = sum;
            }
            __syncthreads();
            uint32_t group = 15, above = 0;
            for (; group > 0 && above + (uint32_t)shared().list[group] < left; --group) above += (uint32_t)shared().list[group];
            uint32_t digit = group * SHARE + SHARE - 1;
            for (; digit > group * SHARE && above + shared().at[digit] < left; --digit) above += shared().at[digit];
            left -= above;
            value |= digit << low;
            high = low;
        }
        return value;
    }
    // The exact k largest: those above the k-th largest value, and of those equal to it the lowest-index ones.  limit: a
    // value that k logits reach.  (Reads the slice at most seven times, nine in rows of up to 64 vectors.  4096 rows of
    // 30522 rising fp32 logits, k = 20: 845 us; 93 where it is not needed.)
    static __device__ void select_exactly(const RowSpan<T>& span, const Slice& s, uint32_t k, uint32_t limit, bool known) {
        if (s.e1 - s.e0 <= k) {
            clear_count();
            elements(span, s, [&](uint32_t order, uint32_t j) {
                if (j < s.e1) append(order, j);
                return true;
            });
            __syncthreads();
            return;
        }
        // (known: limit is the k-th largest if fewer than k logits are above it -- a masked vocabulary)
        if (!known || reaching(span, s, limit + 1) >= k) limit = kth_largest(span, s, k, limit);
        clear_count();
        elements(span, s, [&](uint32_t order, uint32_t j) {
            if (order > limit) append(order, j);
            return true;
        });
        __syncthreads();
        fill_up(span, s, k, limit);
    }
    // The list holds the logits above `limit`, which has no more than k - 1 above it: the lowest-index ones that equal it
    // (behind a mask, among the slice's first ones) complete it to k, as far as there are any.
    static __device__ void fill_up(const RowSpan<T>& span, const Slice& s, uint32_t k, uint32_t limit) {
        const uint32_t t = threadIdx.x, lane = t & 63, above = shared().count;
        if (above >= k) return;
        const uint32_t want = k - above;
        uint32_t have = 0;
        elements(span, s, [&](uint32_t order, uint32_t j) {
            const bool equal = j < s.e1 && order == limit;
            const uint64_t in_wave = __builtin_amdgcn_ballot_w64(equal);
            __syncthreads();
            if (lane == 0) shared().at[t >> 6] = (uint32_t)__builtin_popcountll(in_wave);
            __syncthreads();
            uint32_t at = have + (uint32_t)__builtin_popcountll(in_wave & ((1ull << lane) - 1));
            for (uint32_t w = 0; w < THREADS / 64; ++w) {
                if (w < (t >> 6)) at += shared().at[w];
                have += shared().at[w];
            }
            if (equal && at < want) shared().list[above + at] = composite(order, j);
            return have < want;
        });
        __syncthreads();
        if (t == 0) shared().count = above + (have < want ? have : want);
        __syncthreads();
    }

    // Keeps those of the thread's G vectors from base on that hold a logit from least (> -inf) on; hi: the largest logit.
    // Which of their logits these are is left to sift(), where every thread looks at one.
    template <int G> static __device__ __forceinline__ void meet(const RowSpan<T>& span, const u32x4* raw, float hi, uint32_t base, float least) {
        if (!(hi >= least)) return;
#pragma unroll
        for (int u = 0; u < G; ++u) {
            float x[N];
            LogitVec<T>::unpack(raw[u], x);
            if (G == 1 || largest(x) >= least) {
                const uint32_t at = __hip_atomic_fetch_add(&shared().n_vectors, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                if (at < (uint32_t)VECTORS) {
                    shared().vectors[at] = raw[u];
                    shared().at[at] = span.index(base + u * THREADS + threadIdx.x);
                }
            }
        }
    }
    static __device__ __forceinline__ void sift(float least) {
        __syncthreads();
        const uint32_t n = shared().n_vectors;
        if (n <= (uint32_t)VECTORS)
            for (uint32_t i = threadIdx.x; i < n * N; i += THREADS) {
                const float x = LogitVec<T>::load((const T*)shared().vectors + i);
                if (x >= least) append(order_of(x), shared().at[i / N] + i % N);
            }
        __syncthreads();
    }
    static __device__ __forceinline__ bool overflow() { return shared().n_vectors > (uint32_t)VECTORS || shared().count > (uint32_t)LIST; }
    // A long row's k largest are collected while it is read: a threshold from the threads' first vectors holds for the
    // whole row and lets through about as many times k logits as the row is longer than they are.
    // The value from which logits are let through; NaN, which lets none through, where there are no k logits.  *tie: the
    // threshold itself, if only logits above it are let through (0: those that equal it too).
    static __device__ __forceinline__ float early(float top, bool any, uint32_t k, uint32_t* tie) {
        uint32_t kind;
        const uint32_t limit = threshold(top, any, k, &kind);
        *tie = kind == kCommon ? limit : 0u;
        if (kind == kCommon) return logit_of(limit + 1);
        return limit <= kMaskedOrder ? __builtin_nanf("") : logit_of(limit);
    }

    static __device__ __forceinline__ void edge(const RowSpan<T>& span, const Slice& s, float least) {
        if (s.edge >= 0) {
            const float x = LogitVec<T>::load(span.row + s.edge);
            if (x >= least) append(order_of(x), (uint32_t)s.edge);
        }
    }
    // Few threads and many alternatives: the threshold lets most of a row through, and ranking n logits costs n^2.  One
    // wave finds the k-th largest of the list and keeps those that reach it.  (9240 rows of 365 with 63: 36 us, without
    // this 97.)
    static __device__ __forceinline__ void thin_out(uint32_t k) {
        const uint32_t n = shared().count, t = threadIdx.x;
        if (n <= THIN) return;
        if (THREADS > 64) __syncthreads();   // (all have read the count before the first wave writes it)
        if (t < 64) {
            constexpr int W = (LIST + 63) / 64;
            uint64_t own[W];
#pragma unroll
            for (int i = 0; i < W; ++i) own[i] = i * 64 + t < n ? shared().list[i * 64 + t] : 0ull;
            uint32_t limit = 0;
            for (int bit = 31; bit >= LOW_BIT; --bit) {
                const uint32_t next = limit | (1u << bit);
                uint32_t reach = 0;
#pragma unroll
                for (int i = 0; i < W; ++i)
                    if (i * 64 < (int)n) reach += (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64((uint32_t)(own[i] >> 32) >= next));
                if (reach >= k) limit = next;
                if (reach == k) break;
            }
            uint32_t at = 0;
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const bool keep = (uint32_t)(own[i] >> 32) >= limit && i * 64 + t < n;
                const uint64_t in_wave = __builtin_amdgcn_ballot_w64(keep);
                if (keep) shared().list[at + (uint32_t)__builtin_popcountll(in_wave & ((1ull << t) - 1))] = own[i];
                at += (uint32_t)__builtin_popcountll(in_wave);
            }
            if (t == 0) shared().count = at;
        }
        __syncthreads();
    }
    // Leaves at least the k largest of the slice (all of them, if it has fewer) in the list, in any order, given
    // the threshold of the threads' largest logits.  look(least): meets the thread's vectors, every(least): the same for
    // any least, -inf among them; top: the thread's largest logit; nan: the row holds a NaN or +inf.
    // A mask's value would fill the list: only logits above it are collected then, and it is filled up.  (10 logits left,
    // fp32, k = 20: 2000 rows of 131072 take 160 us, took 945 us with select_exactly(); 4096 rows of 30522 78 and 405.)
    template <typename F, typename E>
    static __device__ __forceinline__ void select(const RowSpan<T>& span, const Slice& s, uint32_t limit, uint32_t kind, float top, bool nan,
                                           uint32_t k, F look, E every) {
        if (!nan) {
            const bool above = kind == kCommon || (kind == kExact && limit == kMaskedOrder);
            const float least = above ? logit_of(limit + 1) : limit <= kMaskedOrder ? -kInf : logit_of(limit);
            if (least == -kInf) every(least);
            else if (top >= least) look(least);
            edge(span, s, least);
            sift(least);
            if (!overflow()) {
                if (above) fill_up(span, s, k, limit);
                return;
            }
        }
        select_exactly(span, s, k, limit, kind != kBetween && !nan);
    }
};

// Rank of every composite of list[0 .. n); those below k go to f(rank, composite).  As many lanes as there are threads
// for share the comparisons of one composite.
template <int THREADS, typename F> __device__ __forceinline__ void ranked(const uint64_t* list, uint32_t n, uint32_t k, F f) {
    uint32_t share = 1;
    while (share < 16 && 2 * share * n <= (uint32_t)THREADS) share *= 2;
    for (uint32_t i0 = 0; i0 < n; i0 += THREADS / share) {
        const uint32_t i = i0 + threadIdx.x / share, part = threadIdx.x % share;
        const uint64_t mine = i < n ? list[i] : ~0ull;
        int rank = 0;
        uint32_t j = part;   // (four reads in flight)
        for (; j + 3 * share < n; j += 4 * share) {
            const uint64_t a = list[j], b = list[j + share], c = list[j + 2 * share], d = list[j + 3 * share];
            rank += (a > mine) + (b > mine) + (c > mine) + (d > mine);
        }
        for (; j < n; j += share) rank += list[j] > mine;
        if (share > 1) rank += __builtin_amdgcn_update_dpp(0, rank, 0xB1, 0xf, 0xf, true);
        if (share > 2) rank += __builtin_amdgcn_update_dpp(0, rank, 0x4E, 0xf, 0xf, true);
        if (share > 4) rank += __builtin_amdgcn_update_dpp(0, rank, 0x141, 0xf, 0xf, true);
        if (share > 8) rank += __builtin_amdgcn_update_dpp(0, rank, 0x140, 0xf, 0xf, true);
        if (part == 0 && i < n && (uint32_t)rank < k) f((uint32_t)rank, mine);
    }
}

struct LogprobParams {
    const void* logits;
    const int32_t* tokens;
    float *logprob, *entropy, *stats, *top_logprobs;
    int32_t* top_ids;
    uint64_t stride;
    uint32_t vocab, n_tokens, top_k;
    float scale, c;
};

// Half the distance of a logit from the reference: the distance itself may pass the largest fp32.
__device__ __forceinline__ float half_distance(float x, float m) { return 0.5f * x - 0.5f * m; }
// ln p of a logit x from a row's statistics; a row without any logit above -inf gives -inf
__device__ __forceinline__ float log_prob(float x, float m, float l, float scale) {
    return l == -kInf ? -kInf : half_distance(x, m) * (2.f * scale) - l * kLn2;
}

// The logits of a row's tokens, one per thread, fetched before the row is read: by the time its sums are known they
// have arrived, and no thread waits for two dependent loads while the others wait for it.
template <typename T, int THREADS> struct NamedLogits {
    static constexpr int ROUNDS = THREADS < (int)kMaxSlots ? (int)kMaxSlots / THREADS : 1;
    uint32_t x[ROUNDS];   // bits
    int32_t id[ROUNDS];   // -1: none
    // (two steps: the loads of the row go between them, so that the wait for the ids is not one for the row)
    __device__ __forceinline__ void load_ids(const int32_t* ids, uint32_t n) {
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const uint32_t i = threadIdx.x + r * THREADS;
            id[r] = -1;
            if (r * THREADS < (int)n && i < n) id[r] = ids[i];
        }
    }
    __device__ __forceinline__ void load_logits(const RowSpan<T>& span, uint32_t vocab) {
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            if ((uint32_t)id[r] >= vocab) id[r] = -1;
            x[r] = 0;
            if (id[r] >= 0) x[r] = LogitVec<T>::bits(span.row + id[r]);
        }
    }
    __device__ __forceinline__ void write(float* logprob, uint32_t n, float m, float l, float scale) const {
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const uint32_t i = threadIdx.x + r * THREADS;
            if (i < n) logprob[i] = id[r] >= 0 ? log_prob(LogitVec<T>::value(x[r]), m, l, scale) : 0.f;
        }
    }
};

template <bool ENTROPY> __device__ __forceinline__ void write_row_sums(const LogprobParams& p, size_t row, const RowSum& r, float l) {
    if (p.stats) { p.stats[2 * row] = r.m; p.stats[2 * row + 1] = l; }
    if (ENTROPY) {
        const float h = (l - r.dot / r.sum) * kLn2;
        p.entropy[row] = l == -kInf || h < 0.f ? 0.f : h;   // (rounding can leave a certain row below zero)
    }
}

template <int THREADS> __device__ __forceinline__ void write_alternatives(const LogprobParams& p, size_t row, const uint64_t* list,
                                                                        uint32_t n, const RowSum& r, float l) {
    ranked<THREADS>(list, n, p.top_k, [&](uint32_t rank, uint64_t c) {
        p.top_ids[row * p.top_k + rank] = (int32_t)~(uint32_t)c;
        p.top_logprobs[row * p.top_k + rank] = log_prob(logit_of((uint32_t)(c >> 32)), r.m, l, p.scale);
    });
}

// Short rows: one work-group per row, held in registers (NV vectors per thread), so that the sums are taken relative to
// the row's maximum and the alternatives are looked up without another read.  8192 rows of 2000 fp32 logits with entropy
// take 14.8 us (4.4 TB/s), with 4 alternatives 19.6; with tens of them the instructions of their search count for more
// than the memory (8000 rows, 64 alternatives: 36 us).
template <typename T, int THREADS, int NV, bool ENTROPY>
__global__ __launch_bounds__(THREADS) void token_logprobs_held_kernel(LogprobParams p) {
    typedef TopSelect<T, THREADS, NV> Top;
    __shared__ float red[2 * THREADS / 64];
    constexpr int N = LogitVec<T>::N;
    const uint32_t t = threadIdx.x, k = p.top_k;
    const size_t row = blockIdx.x;
    const RowSpan<T> span((const T*)p.logits + row * p.stride, p.vocab);
    const Slice s = slice_of(span, p.vocab, 0, 1, 0, t);
    NamedLogits<T, THREADS> named;
    named.load_ids(p.tokens + row * p.n_tokens, p.n_tokens);
    Held<T, THREADS, NV> held;
    held.load(span, s, t);
    named.load_logits(span, p.vocab);
    const bool any = t < s.v1 || s.edge >= 0;
    auto part = [&](int i) {
        constexpr int each = NV / Top::PER;
        uint32_t order = 0;
#pragma unroll
        for (int u = 0; u < each; ++u)
            if (s.v0 + (i * each + u) * THREADS + t < s.v1) {
                float x[N];
                LogitVec<T>::unpack(held.raw[i * each + u], x);
                const uint32_t o = order_of(largest(x));
                order = order > o ? order : o;
            }
        return order;
    };
    auto publish = [&](float hi) { if (k) Top::publish(hi, any, k, part); };
    auto met = [&](float) {
        if (k) Top::find(k);
        return 0.f;
    };
    const RowSum r = held.template sums<ENTROPY, false>(s, t, p.c, red, publish, met);
    const float l = log2f(r.sum);
    if (t == 0) write_row_sums<ENTROPY>(p, row, r, l);
    named.write(p.logprob + row * p.n_tokens, p.n_tokens, r.m, l, p.scale);
    if (k == 0) return;
    if (THREADS == 64) __syncthreads();
    uint32_t kind;
    const uint32_t limit = Top::found(&kind);
    auto look = [&](float from) {
        held.template steps<false>(s, t, [&](auto count, const u32x4* raw, uint32_t base) {
            Top::template meet<decltype(count)::value>(span, raw, largest_of<T, decltype(count)::value>(raw), base, from);
        });
    };
    auto every = [&](float from) {
        held.each(s, t, [&](const float (&x)[N], uint32_t base) { Top::scan(x, span.index(base + t), from); });
    };
    Top::select(span, s, limit, kind, r.top, r.sum != r.sum, k, look, every);
    Top::thin_out(k);
    write_alternatives<THREADS>(p, row, Top::shared().list, Top::shared().count, r, l);
}

// The sums of a streamed slice; with k > 0 its logits from `least` on are collected on the way.
template <typename T, int THREADS, bool ENTROPY>
__device__ __forceinline__ RowSum sum_and_collect(const RowSpan<T>& span, const Slice& s, float c, float* red, uint32_t k, bool any,
                                                  float& least, uint32_t& tie) {
    typedef TopSelect<T, THREADS, 0> Top;
    least = __builtin_nanf("");
    tie = 0;
    auto early = [&](auto first) { if (k) least = Top::early(first(), any, k, &tie); };
    auto meet = [&](auto count, const u32x4* raw, float hi, uint32_t base) {
        Top::template meet<decltype(count)::value>(span, raw, hi, base, least);
    };
    return Streamed<T, THREADS>::template sums<ENTROPY, false>(span, s, threadIdx.x, c, red, early, meet, [](float) { return 0.f; });
}
// At least the k largest in the list.  Where the early threshold let too many through, or none, the row is read again.
template <typename T, int THREADS>
__device__ __forceinline__ void finish_collection(const RowSpan<T>& span, const Slice& s, const RowSum& r, uint32_t k, bool any, float least,
                                                  uint32_t tie) {
    typedef TopSelect<T, THREADS, 0> Top;
    constexpr int N = LogitVec<T>::N;
    const uint32_t t = threadIdx.x;
    const bool nan = r.sum != r.sum;
    if (least == least) Top::edge(span, s, least);
    Top::sift(least);
    if (least == least && !nan && !Top::overflow()) {
        if (tie) Top::fill_up(span, s, k, tie);
        return;
    }
    uint32_t kind = Top::kBetween;
    const uint32_t limit = Top::threshold(r.top, any, k, &kind);
    auto every = [&](float from) {
        Streamed<T, THREADS>::each(span, s, t, [&](const float (&x)[N], uint32_t base) { Top::scan(x, span.index(base + t), from); });
    };
    Top::select(span, s, limit, kind, r.top, nan, k, every, every);
}

// Long rows: one work-group per row, streamed.  8192 rows of 50257 bf16 logits take 126 us (6.5 TB/s), 4096 of 30522 fp32
// with entropy and 5 alternatives 80 us (6.3 TB/s): bound by memory.  With entropy, bf16 rows are bound by instructions
// nearly as much: 4096 of 30522 take 43 us (5.8 TB/s), 53 with 20 alternatives.
template <typename T, int THREADS, bool ENTROPY>
__global__ __launch_bounds__(THREADS, 8) void token_logprobs_stream_kernel(LogprobParams p) {
    typedef TopSelect<T, THREADS, 0> Top;
    __shared__ float red[2 * THREADS / 64];
    const uint32_t t = threadIdx.x, k = p.top_k;
    const size_t row = blockIdx.x;
    const RowSpan<T> span((const T*)p.logits + row * p.stride, p.vocab);
    const Slice s = slice_of(span, p.vocab, 0, 1, 0, t);
    NamedLogits<T, THREADS> named;
    named.load_ids(p.tokens + row * p.n_tokens, p.n_tokens);
    named.load_logits(span, p.vocab);
    const bool any = t < s.v1 || s.edge >= 0;
    float least;
    uint32_t tie;
    const RowSum r = sum_and_collect<T, THREADS, ENTROPY>(span, s, p.c, red, k, any, least, tie);
    const float l = log2f(r.sum);
    if (t == 0) write_row_sums<ENTROPY>(p, row, r, l);
    named.write(p.logprob + row * p.n_tokens, p.n_tokens, r.m, l, p.scale);
    if (k == 0) return;
    finish_collection<T, THREADS>(span, s, r, k, any, least, tie);
    write_alternatives<THREADS>(p, row, Top::shared().list, Top::shared().count, r, l);
}

// Very short rows: 16 lanes a row, so that a wave's instructions serve four rows and every reduction is four DPP moves.
// Up to kShortTop alternatives are taken out one by one, which is what bounds this kernel: 32768 rows of 256 fp32 logits
// take 7.6 us without alternatives (4.5 TB/s) and 14.8 with 4, where a wave for each row takes 14.0 and 24.7.  (8
// alternatives: 20.8 and 24.7; more are left to those.  500 bf16 logits: 21 and 32.)
constexpr uint32_t kShortTop = 8, kShortVecs = 64, kShortRows = 16;

template <int CTRL> __device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <typename V, typename F> __device__ __forceinline__ V over16(V v, F f) {
    v = f(v, dpp<0xB1>(v));
    v = f(v, dpp<0x4E>(v));
    v = f(v, dpp<0x141>(v));
    return f(v, dpp<0x140>(v));
}

template <typename T, bool ENTROPY>
__global__ __launch_bounds__(256) void token_logprobs_short_kernel(LogprobParams p, uint32_t rows) {
    constexpr int N = LogitVec<T>::N, VECS = kShortVecs / 16, E = VECS * N + 1;
    const uint32_t g = threadIdx.x & 15, wanted = blockIdx.x * kShortRows + threadIdx.x / 16;
    const size_t row = wanted < rows ? wanted : rows - 1;   // (lanes past the last row repeat it and write nothing)
    const bool writes = wanted < rows;
    const RowSpan<T> span((const T*)p.logits + row * p.stride, p.vocab);
    const int32_t edge = span.edge(g);
    u32x4 raw[VECS];
#pragma unroll
    for (int u = 0; u < VECS; ++u) raw[u] = u32x4{LogitVec<T>::kMasked, LogitVec<T>::kMasked, LogitVec<T>::kMasked, LogitVec<T>::kMasked};
    if (span.vecs > 0) {
#pragma unroll
        for (int u = 0; u < VECS; ++u) {
            const uint32_t i = g + 16 * u;
            raw[u] = __builtin_nontemporal_load(span.at(0, i < span.vecs ? i : span.vecs - 1));
        }
    }
    uint32_t edge_bits = LogitVec<T>::kMaskedOne;
    if (edge >= 0) edge_bits = LogitVec<T>::bits(span.row + edge);
    float x[E];
#pragma unroll
    for (int u = 0; u < VECS; ++u) {
        if (g + 16 * u >= span.vecs) raw[u] = u32x4{LogitVec<T>::kMasked, LogitVec<T>::kMasked, LogitVec<T>::kMasked, LogitVec<T>::kMasked};
        float v[N];
        LogitVec<T>::unpack(raw[u], v);
#pragma unroll
        for (int j = 0; j < N; ++j) x[u * N + j] = v[j];
    }
    x[E - 1] = LogitVec<T>::value(edge_bits);
    RowSum r;
    r.top = largest(x);
    r.m = over16(r.top, [](float a, float b) { return fmaxf(a, b); });
    r.sum = r.dot = 0.f;
    const float m = r.m == -kInf ? 0.f : r.m;
#pragma unroll
    for (int e = 0; e < E; ++e) add_term<ENTROPY>((x[e] - m) * p.c, r.sum, r.dot);
    const auto plus = [](float a, float b) { return a + b; };
    r.sum = over16(r.sum, plus);
    if (ENTROPY) r.dot = over16(r.dot, plus);
    const float l = log2f(r.sum);
    if (g == 0 && writes) write_row_sums<ENTROPY>(p, row, r, l);
    for (uint32_t i = g; i < p.n_tokens; i += 16) {
        const int32_t id = p.tokens[row * p.n_tokens + i];
        float lp = 0.f;
        if (id >= 0 && (uint32_t)id < p.vocab) lp = log_prob(LogitVec<T>::load(span.row + id), r.m, l, p.scale);
        if (writes) p.logprob[row * p.n_tokens + i] = lp;
    }
    if (p.top_k == 0) return;
    // an element that is not there is below every logit
    uint32_t order[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const bool there = e == E - 1 ? edge >= 0 : g + 16 * (e / N) < span.vecs;
        order[e] = there ? order_of(x[e]) : 0u;
    }
    for (uint32_t k = 0; k < p.top_k; ++k) {
        uint32_t mine = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) mine = mine > order[e] ? mine : order[e];
        const uint32_t best = over16(mine, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
        // the lowest element that has it: this lane's (an edge element may be the row's first ones or its last), then all
        uint32_t at = E, index = 0xffffffffu;
#pragma unroll
        for (int e = E - 2; e >= 0; --e) at = order[e] == best ? e : at;
        if (at != E) index = span.index(g + 16 * (at / N)) + at % N;
        if (order[E - 1] == best && (uint32_t)edge < index) { at = E - 1; index = (uint32_t)edge; }
        const uint32_t own = index;
        index = over16(index, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
        if (own != index) at = E;
#pragma unroll
        for (int e = 0; e < E; ++e) order[e] = at == e ? 0 : order[e];
        if (g == 0 && writes) {
            p.top_ids[row * p.top_k + k] = (int32_t)index;
            p.top_logprobs[row * p.top_k + k] = log_prob(logit_of(best), r.m, l, p.scale);
        }
    }
}

// ---- few long rows --------------------------------------------------------------------------------------------
// Each row is cut into parts with a work-group each.  A part leaves its sums and its own k largest in the workspace; the
// one that arrives last joins them (in the order of the parts) and writes the row, and clears the row's counter.  Records
// go through the memory system's coherent level with device-scope stores and loads; a part waits for its stores before
// it counts itself as arrived.  Bound by latency: one row of 30522 fp32 logits with 5 alternatives takes 8.4 us, 48 of
// 131072 bf16 with 20 13 us (21 by one work-group a row).
constexpr uint32_t kSplitRows = 512, kSplitParts = 64, kSplitThreads = 512;

struct SplitWork {
    uint32_t* counters;   // [kSplitRows], zero between launches
    float* stats;         // [kSplitRows][2], where the caller keeps none
    uint8_t* records;
    uint32_t parts, each, record_bytes;
};

template <typename V> __device__ __forceinline__ void leave(V* p, V v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename V> __device__ __forceinline__ V take(const V* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// Counts this part of `row` as arrived, once all that the work-group has left is there; whether it is the last.
__device__ __forceinline__ bool arrive(const SplitWork& w, size_t row, uint32_t* arrived) {
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    __syncthreads();
    if (threadIdx.x == 0) *arrived = __hip_atomic_fetch_add(w.counters + row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    return *arrived == w.parts - 1;
}
// The row's sums from its parts' ones (m, sum, dot at the start of each record), by one wave, in joined[0 .. 3); clears the
// row's counter.
template <bool ENTROPY>
__device__ __forceinline__ void join_sums(const SplitWork& w, size_t row, const uint8_t* records, float c, float* joined) {
    const uint32_t t = threadIdx.x;
    if (t >= 64) return;
    float m = -kInf, sum = 0.f, dot = 0.f;
    if (t < w.parts) {
        const float* const f = (const float*)(records + t * w.record_bytes);
        m = take(f);
        sum = take(f + 1);
        if (ENTROPY) dot = take(f + 2);
    }
    const float top = wave_max(m);
    if (m != top) {   // from this part's reference to the row's
        const float d = (m - top) * c, f = exp2_fast(d);
        if (ENTROPY) dot = f * (dot + fmaxf(d, -256.f) * sum);
        sum *= f;
    }
    sum = wave_sum(sum);
    if (ENTROPY) dot = wave_sum(dot);
    if (t == 0) {
        joined[0] = top;
        joined[1] = sum;
        joined[2] = dot;
        leave(w.counters + row, 0u);
    }
}

template <typename T, bool ENTROPY>
__global__ __launch_bounds__(kSplitThreads, 4) void token_logprobs_split_kernel(LogprobParams p, SplitWork w) {
    constexpr int THREADS = kSplitThreads;
    typedef TopSelect<T, THREADS, 0> Top;
    typedef Streamed<T, THREADS> Stream;
    __shared__ float red[2 * THREADS / 64];
    __shared__ uint32_t arrived;
    __shared__ float joined[3];
    const uint32_t t = threadIdx.x, k = p.top_k, part = blockIdx.x % w.parts;
    const size_t row = blockIdx.x / w.parts;
    const RowSpan<T> span((const T*)p.logits + row * p.stride, p.vocab);
    const Slice s = slice_of(span, p.vocab, part, w.parts, w.each, t);
    NamedLogits<T, THREADS> named;
    named.load_ids(p.tokens + row * p.n_tokens, p.n_tokens);
    named.load_logits(span, p.vocab);
    const bool any = s.v0 + t < s.v1 || s.edge >= 0;
    float least;
    uint32_t tie;
    RowSum r = sum_and_collect<T, THREADS, ENTROPY>(span, s, p.c, red, k, any, least, tie);
    uint8_t* const records = w.records + row * w.parts * w.record_bytes;
    uint8_t* const record = records + part * w.record_bytes;
    if (t < 3) leave((float*)record + t, t == 0 ? r.m : t == 1 ? r.sum : r.dot);
    if (k) {
        finish_collection<T, THREADS>(span, s, r, k, any, least, tie);
        const uint32_t n = Top::shared().count;
        uint64_t* const best = (uint64_t*)(record + 16);
        ranked<THREADS>(Top::shared().list, n, k, [&](uint32_t rank, uint64_t c) { leave(best + rank, c); });
        for (uint32_t i = n + t; i < k; i += THREADS) leave(best + i, (uint64_t)0);   // (a part of fewer logits)
    }
    if (!arrive(w, row, &arrived)) return;
    join_sums<ENTROPY>(w, row, records, p.c, joined);
    if (k) {
        // At least k of the parts' logits reach the least of their r-th largest ones, r parts >= k: with that as a
        // threshold about two k of the parts k are ranked.
        const uint32_t r = (k + w.parts - 1) / w.parts;
        if (t == 0) Top::shared().count = 0;
        if (t < 64) {
            uint32_t order = 0xffffffffu;
            if (t < w.parts) order = (uint32_t)(take((const uint64_t*)(records + t * w.record_bytes + 16) + r - 1) >> 32);
            order = over16(order, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
            if (t % 16 == 0) Top::shared().at[t / 16] = order;
        }
        __syncthreads();
        uint32_t limit = Top::shared().at[0];
        for (int i = 1; i < 4; ++i) limit = limit < Top::shared().at[i] ? limit : Top::shared().at[i];
        for (uint32_t i = t; i < w.parts * k; i += THREADS) {
            const uint64_t c = take((const uint64_t*)(records + (i / k) * w.record_bytes + 16) + i % k);
            if ((uint32_t)(c >> 32) >= limit) Top::append((uint32_t)(c >> 32), ~(uint32_t)c);
        }
    }
    __syncthreads();
    r.m = joined[0];
    r.sum = joined[1];
    r.dot = joined[2];
    const float l = log2f(r.sum);
    if (t == 0) write_row_sums<ENTROPY>(p, row, r, l);
    named.write(p.logprob + row * p.n_tokens, p.n_tokens, r.m, l, p.scale);
    if (k) write_alternatives<THREADS>(p, row, Top::shared().list, Top::shared().count, r, l);
}

// ---- gradients ------------------------------------------------------------------------------------------------
// Both operators' gradients have one form.  With coefficients c_i on tokens id_i, C = sum_i c_i over the valid ones and
// g the gradient of the entropy H:   dx_j = s ( sum_{i: id_i = j} c_i - C p_j - g p_j (ln p_j + H) ).
struct RowGrad {
    float m, l, c;
    float whole;     // -s C 2^-l
    float ent, H;    // -s g 2^-l, entropy
    __device__ __forceinline__ void set(float m_, float l_, float c_, float minus_s_C, float minus_s_g, float H_) {
        const float inv = exp2_fast(-l_);
        m = m_; l = l_; c = c_; H = H_;
        whole = minus_s_C * inv;
        ent = minus_s_g * inv;
    }
    template <bool ENTROPY> __device__ __forceinline__ float at(float x) const {
        const float t = (x - m) * c, e = exp2_fast(t);
        float d = whole * e;
        if (ENTROPY) d = fmaf(ent * e, fmaf(fmaxf(t, -256.f) - l, kLn2, H), d);
        return d;
    }
};

// The tokens that a row's coefficients belong to, and those coefficients, in shared memory, filled up with id -1 to a
// whole number of fours.  Tokens named more than once are rare but have to add up: a bit per token (its lower 13 bits)
// tells the slots that come second to one, and only tokens that such a slot names are searched for in the whole list.
// (5801 bf16 rows of 3339 logits and 150 slots: 22 us, 58 with every slot searching.)
struct Slots {
    int32_t id[kMaxSlots];
    float coef[kMaxSlots];
    uint32_t seen[256];
    int32_t again[kMaxSlots];
    uint32_t n_again;

    // three steps with a barrier after each: put() every slot, mark() every slot, then the rest of it can be read
    __device__ __forceinline__ void put(uint32_t i, int32_t token) {
        id[i] = token;
        seen[(uint32_t)token >> 5 & 255u] = 0;
    }
    template <int THREADS> __device__ __forceinline__ void finish(uint32_t n) {
        const uint32_t t = threadIdx.x;
        if (n + t < (n + 3) / 4 * 4) {   // (at most three)
            id[n + t] = -1;
            coef[n + t] = 0.f;
        }
        if (t == 0) n_again = 0;
    }
    __device__ __forceinline__ void mark(int32_t token, uint32_t vocab) {
        if ((uint32_t)token >= vocab) return;
        const uint32_t bit = 1u << ((uint32_t)token & 31u);
        const uint32_t before = __hip_atomic_fetch_or(&seen[(uint32_t)token >> 5 & 255u], bit, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        if (before & bit) again[__hip_atomic_fetch_add(&n_again, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP)] = token;
    }
};
// The gradient's entries that tokens name: equal tokens add up in slot order, and the first of them writes the entry.
template <typename T, int THREADS> struct NamedEntries {
    static constexpr uint32_t ROUNDS = THREADS < (int)kMaxSlots ? kMaxSlots / THREADS : 1;
    float value[ROUNDS];
    int32_t id[ROUNDS];   // -1: nothing to write
    // sums of the coefficients of this thread's tokens in elements [e0, e1)
    __device__ __forceinline__ void total(const Slots& slots, uint32_t n, uint32_t e0, uint32_t e1) {
        const uint32_t many = slots.n_again;
#pragma unroll
        for (uint32_t r = 0; r < ROUNDS; ++r) {
            const uint32_t i = threadIdx.x + r * THREADS;
            id[r] = -1;
            value[r] = 0.f;
            if (r * THREADS >= n || i >= n) continue;
            const int32_t mine = slots.id[i];
            if (mine < 0 || (uint32_t)mine < e0 || (uint32_t)mine >= e1) continue;
            bool alone = true, first = true;
            for (uint32_t k = 0; k < many; ++k) alone = alone && slots.again[k] != mine;
            float sum = slots.coef[i];
            if (!alone) {
                sum = 0.f;
#pragma unroll 2
                for (uint32_t k = 0; k < n; k += 4) {
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        const bool same = slots.id[k + j] == mine;
                        sum += same ? slots.coef[k + j] : 0.f;
                        first = first && !(same && k + j < i);
                    }
                }
            }
            if (first) id[r] = mine;
            value[r] = sum;
        }
    }
    // the rest of these entries: their own logits, read before any gradient is written (d may be the logits)
    template <bool ENTROPY> __device__ __forceinline__ void finish(const RowSpan<T>& span, const RowGrad& g, float scale) {
#pragma unroll
        for (uint32_t r = 0; r < ROUNDS; ++r)
            if (id[r] >= 0) value[r] = fmaf(scale, value[r], g.template at<ENTROPY>(LogitVec<T>::load(span.row + id[r])));
    }
    __device__ __forceinline__ void write(T* d) const {
#pragma unroll
        for (uint32_t r = 0; r < ROUNDS; ++r)
            if (id[r] >= 0) LogitVec<T>::store(d + id[r], value[r]);
    }
};

// Writes a slice of a row's gradient but for the entries that tokens name; d may be the logits themselves.  each(f):
// f(x, base) for every vector of the thread.
template <typename T, bool ENTROPY, typename EACH>
__device__ __forceinline__ void write_gradient(const RowSpan<T>& span, const Slice& s, T* d, const RowGrad& g, EACH each) {
    constexpr int N = LogitVec<T>::N;
    const uint32_t t = threadIdx.x;
    const RowSpan<T> to = span.onto(d);
    each([&](float (&x)[N], uint32_t base) {
#pragma unroll
        for (int u = 0; u < N; ++u) x[u] = g.template at<ENTROPY>(x[u]);
        __builtin_nontemporal_store(LogitVec<T>::pack(x), (u32x4*)to.at(base, t));
    });
    if (s.edge >= 0) LogitVec<T>::store(d + s.edge, g.template at<ENTROPY>(LogitVec<T>::load(span.row + s.edge)));
}

// A row that nothing reaches (padding): zeros, whatever its logits hold.
template <typename T, int THREADS> __device__ __forceinline__ void write_zeros(const RowSpan<T>& span, const Slice& s, T* d) {
    const RowSpan<T> to = span.onto(d);
    for (uint32_t base = s.v0; base + threadIdx.x < s.v1; base += THREADS)
        __builtin_nontemporal_store(u32x4{0, 0, 0, 0}, (u32x4*)to.at(base, threadIdx.x));
    if (s.edge >= 0) LogitVec<T>::store(d + s.edge, 0.f);
}

// ---- a teacher's list -----------------------------------------------------------------------------------------
// One wave's view of a teacher's list: the softmax over its used slots.
struct Teacher {
    static constexpr uint32_t ROUNDS = kMaxSlots / 64;
    uint32_t bits[ROUNDS];
    float minus_entropy;   // sum q log2 q
    bool some;             // there is a distribution: a used slot above -inf
    __device__ __forceinline__ void load(const void* z, int as_bf16, size_t first, uint32_t n) {
#pragma unroll
        for (uint32_t r = 0; r < ROUNDS; ++r) {
            const uint32_t i = (threadIdx.x & 63) + 64 * r;
            bits[r] = 0;
            if (64 * r < n && i < n) bits[r] = as_bf16 ? ((const uint16_t*)z)[first + i] : ((const uint32_t*)z)[first + i];
        }
    }
    // q[0 .. n) from the slots' ids; what is past n is left alone
    __device__ __forceinline__ void softmax(const int32_t* ids, int as_bf16, uint32_t n, uint32_t vocab, float c, float* q) {
        const uint32_t lane = threadIdx.x & 63;
        float v[ROUNDS], hi = -kInf;
#pragma unroll
        for (uint32_t r = 0; r < ROUNDS; ++r) {
            const uint32_t i = lane + 64 * r;
            v[r] = -kInf;
            if (64 * r < n && i < n) {
                const int32_t id = ids[i];
                if (id >= 0 && (uint32_t)id < vocab) v[r] = as_bf16 ? bf16_bits_to_f32(bits[r]) : __builtin_bit_cast(float, bits[r]);
            }
            hi = fmaxf(hi, v[r]);
        }
        hi = wave_max(hi);
        float sum = 0.f;
#pragma unroll
        for (uint32_t r = 0; r < ROUNDS; ++r)
            if (64 * r < n && v[r] != -kInf) sum += exp2_fast((v[r] - hi) * c);
        sum = wave_sum(sum);
        const float l = log2f(sum);
        minus_entropy = 0.f;
#pragma unroll
        for (uint32_t r = 0; r < ROUNDS; ++r) {
            const uint32_t i = lane + 64 * r;
            if (64 * r < n && i < n) {
                float qi = 0.f;
                if (v[r] != -kInf) {
                    const float lq = (v[r] - hi) * c - l;
                    qi = exp2_fast(lq);
                    minus_entropy += qi * fmaxf(lq, -256.f);
                }
                q[i] = qi;
            }
        }
        some = !(sum == 0.f);
        minus_entropy = wave_sum(minus_entropy);
    }
};

// ---- gradients from a row's statistics ------------------------------------------------------------------------
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
    uint32_t vocab, n, parts, each;
    int teacher_bf16;
    float scale, c;
};

// One work-group per THREADS * kGradVecs vectors of a row, all read before the first is written.  Bound by memory: 2048
// rows of 50257 fp32 logits against a teacher's 100 take 139 us (5.9 TB/s read and written), 4096 of 30522 bf16 with the
// entropy's term 93 us (5.4 TB/s).  Pieces of 1024 to 4096 vectors differ by a few percent.
constexpr int kGradVecs = 4;
template <typename T, int THREADS, bool ENTROPY, bool TEACHER>
__global__ __launch_bounds__(THREADS) void logit_gradient_kernel(GradParams p) {
    constexpr int NV = kGradVecs;
    __shared__ float red[2 * THREADS / 64];
    __shared__ Slots slots;
    __shared__ uint32_t some_teacher;
    const uint32_t t = threadIdx.x;
    const size_t row = blockIdx.x / p.parts;
    const RowSpan<T> span((const T*)p.logits + row * p.stride, p.vocab);
    const Slice s = slice_of(span, p.vocab, blockIdx.x % p.parts, p.parts, p.each, t);
    T* const d = (T*)p.d_logits + row * p.stride;
    const float m = p.stats[2 * row], l = p.stats[2 * row + 1];
    const float ent = ENTROPY ? -p.scale * p.d_entropy[row] : 0.f, H = ENTROPY ? p.entropy[row] : 0.f;
    const float w = TEACHER ? p.d_loss[row] / p.scale : 0.f;
    const float factor = TEACHER ? 1.f : p.scale;   // (what a teacher's coefficients are multiplied by is in w)
    if (l == -kInf || (TEACHER && w == 0.f)) {
        write_zeros<T, THREADS>(span, s, d);
        return;
    }
    Held<T, THREADS, NV> held;
    NamedEntries<T, THREADS> named;
    float C = 0.f;
    if (TEACHER) {
        Teacher teacher;
        if (t < 64) teacher.load(p.teacher, p.teacher_bf16, row * p.n, p.n);
        for (uint32_t i = t; i < p.n; i += THREADS) slots.put(i, p.ids[row * p.n + i]);
        slots.template finish<THREADS>(p.n);
        held.load(span, s, t);
        __syncthreads();
        for (uint32_t i = t; i < p.n; i += THREADS) slots.mark(slots.id[i], p.vocab);
        if (t < 64) {
            teacher.softmax(slots.id, p.teacher_bf16, p.n, p.vocab, p.c, slots.coef);
            if (t == 0) some_teacher = teacher.some ? 1u : 0u;
        }
        __syncthreads();
        if (!some_teacher) {
            write_zeros<T, THREADS>(span, s, d);
            return;
        }
        C = -w;
        named.total(slots, p.n, s.e0, s.e1);
#pragma unroll
        for (uint32_t r = 0; r < named.ROUNDS; ++r) named.value[r] *= -w;
    } else {
        float any = 0.f;
        for (uint32_t i = t; i < p.n; i += THREADS) {
            const int32_t id = p.ids[row * p.n + i];
            const float v = p.d_logprob[row * p.n + i];
            const bool inside = id >= 0 && (uint32_t)id < p.vocab;
            slots.put(i, id);
            slots.coef[i] = inside ? v : 0.f;
            if (inside) { C += v; any += v != 0.f ? 1.f : 0.f; }
        }
        slots.template finish<THREADS>(p.n);
        __syncthreads();
        if (p.n > 1)
            for (uint32_t i = t; i < p.n; i += THREADS) slots.mark(slots.id[i], p.vocab);
        group_sum<THREADS, true>(C, any, red);
        __syncthreads();
        if (any == 0.f && ent == 0.f) {
            write_zeros<T, THREADS>(span, s, d);
            return;
        }
        held.load(span, s, t);
        named.total(slots, p.n, s.e0, s.e1);
    }
    RowGrad g;
    g.set(m, l, p.c, -factor * C, ent, H);
    named.template finish<ENTROPY>(span, g, factor);
    __syncthreads();
    write_gradient<T, ENTROPY>(span, s, d, g, [&](auto f) { held.each(s, t, f); });
    __syncthreads();
    named.write(d);
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

// cross: sum q (x - m) / 2.  (No logit above -inf: the student gives the teacher's tokens no probability.)
__device__ __forceinline__ float row_loss(const Teacher& teacher, float l, float cross, float scale) {
    return l == -kInf ? kInf : (teacher.minus_entropy + l) * kLn2 / (scale * scale) - cross * (2.f / scale);
}

// One work-group per row, held in registers (NV vectors per thread) or, NV = 0, streamed: the student's sums, the loss,
// and (GRAD) the gradient, for which a held row is not read again.  The teacher's softmax and the logits of its tokens
// are ready by the time the row has arrived; with m, l of the student and q of the teacher the loss is
//   ( sum q ln q + ln2 l ) / s^2 - sum q (x - m) / s.
// With the gradient it reads and writes every logit once, which is what bounds it: 8192 rows of 30522 bf16 logits take
// 185 us (5.4 TB/s), 4096 of 131072 416 us (5.2 TB/s), where a copy reaches 6.2: a compute unit has registers for four
// such rows (one of the long ones), and neither reads nor writes for a row that is between its sums and its gradient.
template <typename T, int THREADS, int NV, bool GRAD>
__global__ __launch_bounds__(THREADS, 4) void distill_kernel(DistillParams p) {
    __shared__ float red[2 * THREADS / 64];
    __shared__ Slots slots;
    __shared__ uint32_t some_teacher;
    const uint32_t t = threadIdx.x;
    const size_t row = blockIdx.x;
    const RowSpan<T> span((const T*)p.logits + row * p.stride, p.vocab);
    const Slice s = slice_of(span, p.vocab, 0, 1, 0, t);
    T* const d = GRAD ? (T*)p.d_logits + row * p.stride : nullptr;
    NamedLogits<T, THREADS> logits;
    Teacher teacher;
    if (t < 64) teacher.load(p.teacher, p.teacher_bf16, row * p.n, p.n);
    logits.load_ids(p.ids + row * p.n, p.n);
    float used = 0.f;
#pragma unroll
    for (int r = 0; r < logits.ROUNDS; ++r) {
        const uint32_t i = t + r * THREADS;
        if (i < p.n) slots.put(i, logits.id[r]);
        if ((uint32_t)logits.id[r] < p.vocab) used = 1.f;
    }
    slots.template finish<THREADS>(p.n);
    used = group_max<THREADS>(used, red, []() {});
    if (used == 0.f) {   // no slot (padding): the logits are not read
        if (t == 0) {
            p.row_loss[row] = 0.f;
            if (p.stats) { p.stats[2 * row] = -kInf; p.stats[2 * row + 1] = -kInf; }
        }
        if (GRAD) write_zeros<T, THREADS>(span, s, d);
        return;
    }
    if (GRAD) {
#pragma unroll
        for (int r = 0; r < logits.ROUNDS; ++r) slots.mark(logits.id[r], p.vocab);
    }
    logits.load_logits(span, p.vocab);
    NamedEntries<T, THREADS> named;
    // (called when the maximum is known: q is complete)
    auto met = [&](float m) {
        float cross = 0.f;
#pragma unroll
        for (int r = 0; r < logits.ROUNDS; ++r) {
            const uint32_t i = t + r * THREADS;
            const float q = i < p.n ? slots.coef[i] : 0.f;
            if (!(q <= 0.f)) cross += q * half_distance(LogitVec<T>::value(logits.x[r]), m);
        }
        if (GRAD) named.total(slots, p.n, 0, p.vocab);
        return cross;
    };
    auto softmax = [&]() {
        if (t >= 64) return;
        teacher.softmax(slots.id, p.teacher_bf16, p.n, p.vocab, p.c, slots.coef);
        if (t == 0) some_teacher = teacher.some ? 1u : 0u;
    };
    Held<T, THREADS, NV ? NV : 1> held;
    RowSum r;
    if (NV) {
        held.load(span, s, t);
        softmax();
        r = held.template sums<false, true>(s, t, p.c, red, [](float) {}, met);
    } else {
        softmax();
        r = Streamed<T, THREADS>::template sums<false, true>(span, s, t, p.c, red, [](auto) {}, [](auto, const u32x4*, float, uint32_t) {}, met);
    }
    const float l = log2f(r.sum);
    const bool some = some_teacher != 0;
    if (t == 0) {
        p.row_loss[row] = some ? row_loss(teacher, l, r.dot, p.scale) : 0.f;
        if (p.stats) { p.stats[2 * row] = r.m; p.stats[2 * row + 1] = l; }
    }
    if (!GRAD) return;
    const float w = p.d_loss[row] / p.scale;   // (d_loss / scale^2, the coefficients' size, may pass the largest fp32)
    if (!some || w == 0.f || l == -kInf) {
        write_zeros<T, THREADS>(span, s, d);
        return;
    }
    RowGrad g;
    g.set(r.m, l, p.c, w, 0.f, 0.f);
#pragma unroll
    for (uint32_t i = 0; i < named.ROUNDS; ++i)
        if (named.id[i] >= 0) named.value[i] = fmaf(-w, named.value[i], g.template at<false>(LogitVec<T>::value(logits.x[i])));
    if (!NV) __syncthreads();   // (a streamed row is read again, its named logits have been)
    write_gradient<T, false>(span, s, d, g, [&](auto f) {
        if (NV) held.each(s, t, f);
        else Streamed<T, THREADS>::each(span, s, t, f);
    });
    __syncthreads();
    named.write(d);
}

// Few long rows: the sums and the loss, each row cut over several work-groups.
template <typename T> __global__ __launch_bounds__(kSplitThreads, 8) void distill_split_kernel(DistillParams p, SplitWork w) {
    constexpr int THREADS = kSplitThreads;
    __shared__ float red[2 * THREADS / 64];
    __shared__ Slots slots;
    __shared__ uint32_t arrived;
    __shared__ float joined[3];
    const uint32_t t = threadIdx.x, part = blockIdx.x % w.parts;
    const size_t row = blockIdx.x / w.parts;
    const RowSpan<T> span((const T*)p.logits + row * p.stride, p.vocab);
    const Slice s = slice_of(span, p.vocab, part, w.parts, w.each, t);
    NamedLogits<T, THREADS> logits;
    Teacher teacher;
    if (t < 64) teacher.load(p.teacher, p.teacher_bf16, row * p.n, p.n);
    logits.load_ids(p.ids + row * p.n, p.n);
    float used = 0.f;
    if (t < p.n) slots.put(t, logits.id[0]);
    if ((uint32_t)logits.id[0] < p.vocab) used = 1.f;
    used = group_max<THREADS>(used, red, []() {});
    if (used == 0.f) {
        if (t == 0 && part == 0) {
            p.row_loss[row] = 0.f;
            p.stats[2 * row] = p.stats[2 * row + 1] = -kInf;
        }
        return;
    }
    logits.load_logits(span, p.vocab);
    RowSum r = Streamed<T, THREADS>::template sums<false, false>(span, s, t, p.c, red, [](auto) {}, [](auto, const u32x4*, float, uint32_t) {},
                                                                [](float) { return 0.f; });
    uint8_t* const records = w.records + row * w.parts * w.record_bytes;
    if (t < 2) leave((float*)(records + part * w.record_bytes) + t, t == 0 ? r.m : r.sum);
    if (!arrive(w, row, &arrived)) return;
    join_sums<false>(w, row, records, p.c, joined);
    if (t < 64) teacher.softmax(slots.id, p.teacher_bf16, p.n, p.vocab, p.c, slots.coef);
    __syncthreads();
    const float m = joined[0], l = log2f(joined[1]);
    const float q = t < p.n ? slots.coef[t] : 0.f;
    float cross = 0.f, unused = 0.f;
    if (!(q <= 0.f)) cross = q * half_distance(LogitVec<T>::value(logits.x[0]), m == -kInf ? 0.f : m);
    group_sum<THREADS, false>(cross, unused, red);
    if (t == 0) {
        p.row_loss[row] = teacher.some ? row_loss(teacher, l, cross, p.scale) : 0.f;
        p.stats[2 * row] = m;
        p.stats[2 * row + 1] = l;
    }
}

// How a row is spread over a work-group: threads, and vectors per thread held in registers (0: streamed).  Fewer threads
// wait less for each other, as long as enough rows fit a compute unit.  8192 bf16 rows with their gradient, us: 2000
// logits 20 at {64, 4} and 33 at {256, 4}; 4000: 30 at {64, 8}, 31 at {128, 8}, 33 at {256, 4}; 6000: 43 at {128, 8}, 45
// at {256, 4}; 16000: 99 at {256, 8}, 107 at {512, 8}, 154 at {1024, 8}; 30522: 188 at {512, 8}, 196 at {256, 16}.  4096
// rows of 64000: 186 at {512, 16}, 192 at {1024, 8}, 231 at {1024, 12}, 259 at {1024, 0}, where the row is read twice; of
// 96000: 288 at {512, 24}, 321 at {1024, 12}; of 131072: 418 at {1024, 16}, 423 at {512, 32}.
// Without the gradient nothing needs to be kept, and long rows are streamed.
struct RowShape { int threads, vecs; };
static inline RowShape distill_shape(uint32_t vocab, int dtype, bool gradient) {
    const uint32_t vecs = vocab / (dtype == SFB_BF16 ? 8u : 4u);
    if (vecs <= 64) return {64, 1};
    if (vecs <= 256) return {64, 4};
    if (vecs <= 512) return {64, 8};
    if (vecs <= 1024) return {128, 8};
    if (!gradient) return {512, 0};
    if (vecs <= 2048) return {256, 8};
    if (vecs <= 4096) return {512, 8};
    if (vecs <= 8192) return {512, 16};
    if (vecs <= 12288) return {512, 24};
    if (vecs <= 16384) return {1024, 16};
    return {1024, 0};
}

// Parts of each row of a launch that would otherwise leave most of the device idle: about `groups` work-groups in all, of
// at least 1024 vectors each, or up to 512 where rows would otherwise be halved at most and 8192 are left each.  With 20
// alternatives, us: 48 rows of 16384 vectors 12.4 as 240 groups, 13.6 as 480, 15 as 720, 19.5 whole; 200 of 32768 27 as
// 400, 45 whole; 100 of them 18 as 500, 22 as 200; 200 of 6282 15.6 as 400, 11.8 whole.  parts = 0: no workspace, or too
// many rows.
static inline SplitWork split_rows(void* workspace, uint64_t rows, uint32_t vecs, uint32_t k, uint32_t groups) {
    SplitWork w{};
    if (!workspace || rows > kSplitRows) return w;
    uint32_t parts = groups / (uint32_t)rows;
    if (parts > vecs / 1024) parts = vecs / 1024;
    const uint32_t more = 512 / (uint32_t)rows, longer = vecs / 8192;
    if (parts <= 2 && parts < more && parts < longer) parts = more < longer ? more : longer;
    if (parts > kSplitParts) parts = kSplitParts;
    if (k && parts > 512 / k) parts = 512 / k;   // (the parts' alternatives fit one list)
    if (parts < 1) parts = 1;
    w.parts = parts;
    w.each = (vecs + parts - 1) / parts;
    w.record_bytes = 16 + (k * 8 + 15) / 16 * 16;
    w.counters = (uint32_t*)workspace;
    w.stats = (float*)workspace + kSplitRows;
    w.records = (uint8_t*)workspace + 3 * kSplitRows * sizeof(uint32_t);
    return w;
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
// Whether a gradient's rows are launched twice, cut for the loss and then for the gradient, instead of each by one
// work-group that keeps it.  bf16 rows: 20 of 8125 vectors 12.6 us cut and 11.7 whole, 20 of 12500 13.6 and 16.3, 100 of
// 12500 18.5 and 18.0, 500 of 12500 58 and 45; rows past 16384 vectors, which no work-group holds (fp32): 300 of 32768 85
// and 102, 4 of them 11 and 21.
static inline bool loss_first(uint64_t rows, uint32_t vecs) { return vecs > 16384 || (vecs > 8192 && rows <= 64); }

// A launch has fewer than 2^32 threads.
static inline bool too_many(uint64_t groups, uint32_t threads) { return groups * threads > 0xffffffffull; }
static inline bool misaligned4(const void* a, const void* b = nullptr, const void* c = nullptr, const void* d = nullptr) {
    return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c | (uintptr_t)d) & 3u) != 0;
}

}  // namespace sfb

using namespace sfb;

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
    const uint32_t vecs = vocab / (dtype == SFB_BF16 ? 8u : 4u);
    const SplitWork w = split_rows(workspace, rows, vecs, top_k, 256);
    // Rows that one or two waves hold, else streamed.  8192 fp32 rows with 4 alternatives, us: 1000 logits 14 at 64 x 4, 23
    // at 256 x 4, 43 streamed by 512 threads; 2000: 20 at 64 x 8 and at 128 x 8, 25 at 256 x 4; 4000: 29 at 128 x 8, 32 at
    // 256 x 4, 33 streamed by 256 threads, 49 by 512.  Alternatives of streamed rows cost less with fewer threads until
    // the rows are long: 4096 bf16 rows of 30522 with 20 53 by 256 threads and 58 by 512, without 45 and 44; 4096 fp32
    // ones 89 and 85.
    const bool is_short = vecs <= kShortVecs && top_k <= kShortTop;
    if (too_many(rows, is_short ? 256 / kShortRows : vecs <= 512 ? 64 : vecs <= 1024 ? 128 : 512)) return SFB_ERR_SHAPE;
    const dim3 grid((uint32_t)rows);
#define SFB_LP_AS(T, ENT)                                                                                              \
    do {                                                                                                               \
        if (w.parts > 1)                                                                                               \
            token_logprobs_split_kernel<T, ENT><<<dim3((uint32_t)rows * w.parts), kSplitThreads, 0, s>>>(p, w);        \
        else if (is_short)                                                                                             \
            token_logprobs_short_kernel<T, ENT><<<dim3((uint32_t)((rows + kShortRows - 1) / kShortRows)), 256, 0, s>>>(p, (uint32_t)rows); \
        else if (vecs <= 64) token_logprobs_held_kernel<T, 64, 1, ENT><<<grid, 64, 0, s>>>(p);                         \
        else if (vecs <= 256) token_logprobs_held_kernel<T, 64, 4, ENT><<<grid, 64, 0, s>>>(p);                        \
        else if (vecs <= 512) token_logprobs_held_kernel<T, 64, 8, ENT><<<grid, 64, 0, s>>>(p);                        \
        else if (vecs <= 1024) token_logprobs_held_kernel<T, 128, 8, ENT><<<grid, 128, 0, s>>>(p);                     \
        else if (top_k && vecs <= 4096) token_logprobs_stream_kernel<T, 256, ENT><<<grid, 256, 0, s>>>(p);             \
        else token_logprobs_stream_kernel<T, 512, ENT><<<grid, 512, 0, s>>>(p);                                        \
    } while (0)
#define SFB_LP(T)                        \
    do {                                 \
        if (entropy) SFB_LP_AS(T, true); \
        else SFB_LP_AS(T, false);        \
    } while (0)
    if (dtype == SFB_F32) SFB_LP(float);
    else SFB_LP(__bf16);
#undef SFB_LP_AS
#undef SFB_LP
    return launch_status();
}

static int launch_gradient(hipStream_t s, GradParams& p, int dtype, uint64_t rows, bool entropy, bool teacher) {
    const uint32_t vecs = p.vocab / (dtype == SFB_BF16 ? 8u : 4u);
    // (a row by one wave: 15347 rows of 833 fp32 logits, loss and gradient, 35 us; 50 by four.  8000 of 1500: 38 and 36)
    const uint32_t threads = vecs <= 256 ? 64 : 256;
    p.each = threads * kGradVecs;
    p.parts = vecs == 0 ? 1 : (vecs + p.each - 1) / p.each;
    if (too_many(rows * p.parts, threads)) return SFB_ERR_SHAPE;
    const dim3 grid((uint32_t)(rows * p.parts));
    clear_stale_error();
#define SFB_GR_AS(T, TH)                                                                               \
    do {                                                                                               \
        if (teacher) logit_gradient_kernel<T, TH, false, true><<<grid, TH, 0, s>>>(p);                 \
        else if (entropy) logit_gradient_kernel<T, TH, true, false><<<grid, TH, 0, s>>>(p);            \
        else logit_gradient_kernel<T, TH, false, false><<<grid, TH, 0, s>>>(p);                        \
    } while (0)
#define SFB_GR(T)                              \
    do {                                       \
        if (threads == 64) SFB_GR_AS(T, 64);   \
        else SFB_GR_AS(T, 256);                \
    } while (0)
    if (dtype == SFB_F32) SFB_GR(float);
    else SFB_GR(__bf16);
#undef SFB_GR
#undef SFB_GR_AS
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
    const uint32_t vecs = vocab / (dtype == SFB_BF16 ? 8u : 4u);
    const SplitWork w = split_rows(workspace, rows, vecs, 0, 512);
    if (d_logits ? w.parts > 0 && loss_first(rows, vecs) : w.parts > 1) {
        if (!stats) p.stats = w.stats;
        const dim3 parts((uint32_t)rows * w.parts);
        if (dtype == SFB_F32) distill_split_kernel<float><<<parts, kSplitThreads, 0, s>>>(p, w);
        else distill_split_kernel<__bf16><<<parts, kSplitThreads, 0, s>>>(p, w);
        const int status = launch_status();
        if (status || !d_logits) return status;
        GradParams g{};
        g.logits = logits; g.d_logits = d_logits; g.ids = teacher_ids; g.stats = p.stats; g.teacher = teacher_logits;
        g.teacher_bf16 = p.teacher_bf16; g.d_loss = d_loss; g.stride = row_stride; g.vocab = vocab; g.n = slots;
        g.scale = scale; g.c = p.c;
        return launch_gradient(s, g, dtype, rows, false, true);
    }
    const RowShape shape = distill_shape(vocab, dtype, d_logits != nullptr);
    if (too_many(rows, (uint32_t)shape.threads)) return SFB_ERR_SHAPE;
    const dim3 grid((uint32_t)rows);
#define SFB_DL_AS(T, GRAD)                                                                                         \
    do {                                                                                                           \
        if (shape.threads == 64 && shape.vecs == 1) distill_kernel<T, 64, 1, GRAD><<<grid, 64, 0, s>>>(p);         \
        else if (shape.threads == 64 && shape.vecs == 4) distill_kernel<T, 64, 4, GRAD><<<grid, 64, 0, s>>>(p);    \
        else if (shape.threads == 64) distill_kernel<T, 64, 8, GRAD><<<grid, 64, 0, s>>>(p);                       \
        else if (shape.threads == 128) distill_kernel<T, 128, 8, GRAD><<<grid, 128, 0, s>>>(p);                    \
        else if (!GRAD) distill_kernel<T, 512, 0, false><<<grid, 512, 0, s>>>(p);                                  \
        else if (shape.threads == 256) distill_kernel<T, 256, 8, true><<<grid, 256, 0, s>>>(p);                    \
        else if (shape.vecs == 8) distill_kernel<T, 512, 8, true><<<grid, 512, 0, s>>>(p);                         \
        else if (shape.threads == 512 && shape.vecs == 16) distill_kernel<T, 512, 16, true><<<grid, 512, 0, s>>>(p); \
        else if (shape.vecs == 24) distill_kernel<T, 512, 24, true><<<grid, 512, 0, s>>>(p);                       \
        else if (shape.vecs == 16) distill_kernel<T, 1024, 16, true><<<grid, 1024, 0, s>>>(p);                     \
        else distill_kernel<T, 1024, 0, true><<<grid, 1024, 0, s>>>(p);                                            \
    } while (0)
#define SFB_DL(T)                         \
    do {                                  \
        if (d_logits) SFB_DL_AS(T, true); \
        else SFB_DL_AS(T, false);         \
    } while (0)
    if (dtype == SFB_F32) SFB_DL(float);
    else SFB_DL(__bf16);
#undef SFB_DL_AS
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
