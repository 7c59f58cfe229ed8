// Softmax statistics of [N, V] logits and what is read off them, one pass over the logits:
//   token_logprobs  log probability of a given id, entropy, log-sum-exp and the top alternatives of each row, and the gradient of the first three
//   distill_topk    Kullback-Leibler divergence from a teacher's top entries (CategoricalCrossEntropy over soft targets,
//                   tf/losses/listwise.py:38-52, where the targets are few of V), and its gradient
//
// With z = l / T, m = max l, c = log2(e) / T:  s = sum 2^((l - m) c),  log p = (l - m) / T - ln s,  H = ln2 (log2 s - u / s) with
// u = sum 2^t t, t = (l - m) c.  A thread keeps a running maximum and rescales its sums when it rises; sums are fp32.  All kernels are
// bound by reading the logits (and writing the gradient): 16-byte loads at whatever address a row starts, several in flight a thread.
//
// Masked entries (-inf) have p = 0.  A row with nothing left has log p = -inf, entropy 0 and no gradient.  NaN or +inf makes a row's values NaN.
#include "mh_lowp.h"

#include <type_traits>

namespace {

constexpr float LN2 = 0.693147180559945309f;
// The pass works with l c up to a magnitude of 2^28 (see Run).  A thread's running maximum starts at -2^28 / c: a row whose entries all lie below (masks
// of the type's lowest value) comes out with a sum under 1, where the largest entry alone gives 1; one with an entry beyond 2^29 / c is marked.
// Both are summed again against their true maximum.
constexpr float FAR = 0x1p28f;
constexpr float INF = __builtin_inff();
constexpr int TOP_MOST = 256;        // most alternatives, and teacher entries, of a row
// stretches of a row (or part) whose largest entry LDS holds, in a workgroup of NT threads
template <int NT>
constexpr int buckets() {
    return NT == 256 ? 1024 : 4096;
}
constexpr int CAND = 2048;           // candidates of a row (or part of one) that LDS holds
constexpr int JOIN_MOST = 16 * 512;  // candidates of all parts of a row that the joining kernel holds in registers
constexpr int TAIL_CHUNK = 1 << 18;  // columns of a part whose membership bits lie in LDS (32 KB)

struct Sum {
    float m, s, u;  // maximum, sum 2^t, sum 2^t t with t = (l - m) c
};

__device__ __forceinline__ float ex2(float t) { return __builtin_amdgcn_exp2f(t); }

// a's sums relative to the larger maximum m (>= a.m); the clamp keeps 0 * (d s) from being 0 * inf and loses nothing: 2^-200 is 0
__device__ __forceinline__ void sum_to(Sum& a, float m, float c) {
    const float d = fmaxf((a.m - m) * c, -200.f), f = ex2(d);
    a.u = f * fmaf(d, a.s, a.u);
    a.s *= f;
    a.m = m;
}
__device__ __forceinline__ Sum sum_join(Sum a, Sum b, float c) {
    const float m = fmaxf(a.m, b.m);
    sum_to(a, m, c);
    sum_to(b, m, c);
    return Sum{m, a.s + b.s, a.u + b.u};
}
// Reductions over a wavefront by data-parallel moves (a few cycles each, where a shuffle goes through LDS): within rows of 16 lanes, row 0 into 1 and 2
// into 3, rows 0-1 into 3; lane 63 has it.
template <int CTRL, int ROWS>
__device__ __forceinline__ float moved(float other, float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(other), __float_as_int(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float of_last(float v) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63)); }
__device__ __forceinline__ float max_wave(float v) {
    v = fmaxf(v, moved<0x111, 0xf>(v, v));
    v = fmaxf(v, moved<0x112, 0xf>(v, v));
    v = fmaxf(v, moved<0x114, 0xf>(v, v));
    v = fmaxf(v, moved<0x118, 0xf>(v, v));
    v = fmaxf(v, moved<0x142, 0xa>(v, v));
    v = fmaxf(v, moved<0x143, 0xc>(v, v));
    return of_last(v);
}
__device__ __forceinline__ float add_wave(float v) {
    v += moved<0x111, 0xf>(0.f, v);
    v += moved<0x112, 0xf>(0.f, v);
    v += moved<0x114, 0xf>(0.f, v);
    v += moved<0x118, 0xf>(0.f, v);
    v += moved<0x142, 0xa>(0.f, v);
    v += moved<0x143, 0xc>(0.f, v);
    return of_last(v);
}
__device__ __forceinline__ double add_wave(double v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ Sum sum_wave(Sum a, float c) {
    sum_to(a, max_wave(a.m), c);
    return Sum{a.m, add_wave(a.s), add_wave(a.u)};
}
// Over the first NT threads of a workgroup; every thread of it takes part in the barriers and has the result.
template <int NT>
__device__ __forceinline__ Sum sum_block(Sum a, float c, Sum* red) {
    a = sum_wave(a, c);
    __syncthreads();
    if ((threadIdx.x & 63) == 0 && threadIdx.x < NT) red[threadIdx.x >> 6] = a;
    __syncthreads();
    float m = red[0].m;
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) m = fmaxf(m, red[w].m);
    Sum t = {m, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        Sum b = red[w];
        sum_to(b, m, c);
        t.s += b.s;
        t.u += b.u;
    }
    return t;
}
template <int NT>
__device__ __forceinline__ float max_block(float v, float* red) {
    v = max_wave(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0 && threadIdx.x < NT) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) v = fmaxf(v, red[w]);
    return v;
}
// the sum over the wavefronts of a number that each knows; two sets of places in turn: one barrier a count
template <int NT>
__device__ __forceinline__ int count_block(int of_wave, int* red, int& phase) {
    int* r = red + (phase ^= 1) * (NT / 64);
    if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = of_wave;
    __syncthreads();
    int n = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) n += r[w];
    return n;
}
__device__ __forceinline__ int lanes(bool p) { return __popcll(__ballot(p)); }

// The sums of a thread while it reads: t = l c - B in one fused operation, B the rounded product m c.  What B lacks of m c -- 16 at most below 2^29 --
// is put right once, at the end, exactly: fma(m, c, -B) is what the rounding took.  The step from one B to the next takes the rounded products too:
// fused with its subtraction, B - most c would miss what the later terms are measured from by as much as B lacks.
struct Run {
    float m, B, s = 0.f, u = 0.f;
    __device__ __forceinline__ explicit Run(float c) : m(-FAR / c), B(m * c) {}
    template <bool ENT, int N>
    __device__ __forceinline__ void take(const float (&v)[N], float most, float c) {
        if (most > m) {
#pragma clang fp contract(off)
            const float nb = most * c, d = fmaxf(B - nb, -200.f), f = ex2(d);
            if (ENT) u = f * fmaf(d, s, u);
            s *= f;
            m = most;
            B = nb;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float t = fmaf(v[i], c, -B), e = ex2(t);
            s += e;
            if (ENT) u = fmaf(e, fmaxf(t, -200.f), u);  // 0 * -inf is 0 here; a NaN stays one through e
        }
    }
    __device__ __forceinline__ Sum sum(float c) const {
        const float d = fmaf(m, c, -B), f = ex2(-d);
        return Sum{m, s * f, f * fmaf(-d, s, u)};
    }
};

// a vector of -inf
__device__ __forceinline__ uint4 all_masked(const float*) { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
__device__ __forceinline__ uint4 all_masked(const lp_bf16*) { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
__device__ __forceinline__ uint4 all_masked(const lp_f16*) { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }

template <int N>
__device__ __forceinline__ float most_of(const float (&v)[N]) {
    float a = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) a = fmaxf(a, v[i]);
    return a;
}

// f(values, index of the first) over the n entries at x, in vectors and, at the end, single entries (the others of that call -inf)
template <int NT, typename T, typename F>
__device__ __forceinline__ void each_entry(const T* x, int n, F f) {
    constexpr int VE = lp_vec<T>::N;
    const int nv = n / VE;
    if (threadIdx.x >= NT) return;
    for (int v = threadIdx.x; v < nv; v += NT) {
        float a[VE];
        lp_unpack(lp_load16(x + (int64_t)v * VE), a, x);
        f(a, v * VE);
    }
    if (threadIdx.x < n - nv * VE) {
        float a[VE];
#pragma unroll
        for (int i = 1; i < VE; ++i) a[i] = -INF;
        a[0] = lp_float(x[nv * VE + threadIdx.x]);
        f(a, nv * VE + threadIdx.x);
    }
}

// masks the entries of vector v whose bit is set
template <int VE>
__device__ __forceinline__ void mask_values(float (&a)[VE], const uint32_t* bits, int v) {
    const uint32_t w = VE == 8 ? (bits[v >> 2] >> (8 * (v & 3))) & 255u : (bits[v >> 3] >> (4 * (v & 7))) & 15u;
    if (w) {
#pragma unroll
        for (int i = 0; i < VE; ++i)
            if (w >> i & 1) a[i] = -INF;
    }
}

// The sums over the n entries at x, read by the first NT threads.  SKIP: entries whose bit is set in `skip` do
// not count.  TOP: bucket[v >> shift] receives the largest entry of each vector (shift = 0) or of eight neighbouring ones, 128 bytes (shift = 3); past
// the last bucket they start over at the first, and the same threads come by: their number is a multiple of a round's.
template <int NT, bool ENT, bool SKIP, bool TOP, typename T>
__device__ __forceinline__ Sum read_sums(const T* x, int n, float c, const uint32_t* skip, float* bucket, int shift, Sum* red) {
    constexpr int VE = lp_vec<T>::N, U = 4;
    Run r(c);
    float most = -INF;
    const int nv = n / VE;
    int v = threadIdx.x < NT ? threadIdx.x : (nv | 7) + 1;
    auto batch = [&](const uint4 (&w)[U]) {
        float a[U * VE];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            float b[VE];
            lp_unpack(w[j], b, x);
            if (SKIP && v + j * NT < nv) mask_values(b, skip, v + j * NT);
            if (TOP) {
                float q = most_of(b);
                if (shift) {
                    q = fmaxf(q, moved<0xb1, 0xf>(q, q));   // lanes 1 0 3 2
                    q = fmaxf(q, moved<0x4e, 0xf>(q, q));   // 2 3 0 1
                    q = fmaxf(q, moved<0x141, 0xf>(q, q));  // 7 6 .. 0
                }
                if (v + j * NT < nv && (!shift || (threadIdx.x & 7) == 0)) {
                    const int at = (v + j * NT) >> shift;
                    float* b = bucket + (at & (buckets<NT>() - 1));
                    *b = at < buckets<NT>() ? q : fmaxf(q, *b);
                }
            }
#pragma unroll
            for (int i = 0; i < VE; ++i) a[j * VE + i] = b[i];
        }
        const float b = most_of(a);
        most = fmaxf(most, b);
        r.template take<ENT>(a, b, c);
    };
    // eight lanes go together, so that one of them can speak for a bucket
    for (; (v | 7) + (U - 1) * NT < nv; v += U * NT) {
        uint4 w[U];
#pragma unroll
        for (int j = 0; j < U; ++j) w[j] = lp_load16(x + (int64_t)(v + j * NT) * VE);
        batch(w);
    }
    if ((v & ~7) < nv) {  // the last vectors, together as well
        uint4 w[U];
#pragma unroll
        for (int j = 0; j < U; ++j) w[j] = v + j * NT < nv ? lp_load16(x + (int64_t)(v + j * NT) * VE) : all_masked(x);
        batch(w);
    }
    if (threadIdx.x < n - nv * VE) {  // fewer than a vector: never the extra wavefront
        const int i = nv * VE + threadIdx.x;
        float a[1] = {lp_float(x[i])};
        if (SKIP && (skip[i >> 5] >> (i & 31) & 1)) a[0] = -INF;
        most = fmaxf(most, a[0]);
        r.template take<ENT>(a, a[0], c);
    }
    const bool beyond = __syncthreads_or(!(r.B < 2.f * FAR));
    Sum t = sum_block<NT>(r.sum(c), c, red);
    if (t.s < 0.5f || beyond) {
        t = Sum{max_block<NT>(most, reinterpret_cast<float*>(red)), 0.f, 0.f};
        if (t.m == -INF) return t;
        Sum a = {t.m, 0.f, 0.f};
        each_entry<NT>(x, n, [&](const float(&l)[VE], int at) {
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                if (SKIP && at + i < n && (skip[(at + i) >> 5] >> ((at + i) & 31) & 1)) continue;
                const float d = (l[i] - t.m) * c, e = ex2(d);
                a.s += e;
                a.u = fmaf(e, fmaxf(d, -200.f), a.u);
            }
        });
        t = sum_block<NT>(a, c, red);
    }
    return t;
}

// ---- top alternatives ------------------------------------------------------------------------------------------------------------------
// An entry's key orders by value, then by place, the lowest first; places of -inf and NaN have none.
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __float_as_uint(v);
    return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k); }
constexpr uint32_t KEY_NONE = 0x007fffffu;  // the key of -inf
__device__ __forceinline__ uint64_t key_at(float v, int at) {
    return (v > -INF) ? (uint64_t)key_of(v + 0.f) << 32 | (uint32_t)~at : 0;  // + 0: -0 and 0 are one value
}

// The largest threshold found, from the high bits on, that at least k keys reach; ends as soon as no more than `most` do.
template <typename C>
__device__ __forceinline__ uint64_t key_threshold(int k, int most, C count) {
    uint64_t t = 0;
    for (int b = 63; b >= 0; --b) {
        const uint64_t next = t | (uint64_t)1 << b;
        const int n = count(next);
        if (n >= k) {
            t = next;
            if (n <= most) break;
        }
    }
    return t;
}

// how many of n keys are larger: keys[n], if n is odd, is 0
__device__ __forceinline__ int place_of(uint64_t key, const uint64_t* keys, int n) {
    typedef uint64_t two __attribute__((ext_vector_type(2)));
    int place = 0;
#pragma unroll 8
    for (int i = 0; i < n; i += 2) {
        const two v = *reinterpret_cast<const two*>(keys + i);
        place += (v[0] > key ? 1 : 0) + (v[1] > key ? 1 : 0);
    }
    return place;
}

template <int NT>
struct TopLds {
    __attribute__((aligned(16))) uint64_t cand[CAND + 2];
    union {
        float most[buckets<NT>()];     // while the row is read
        uint16_t list[buckets<NT>()];  // the buckets to read again
    };
    uint32_t low;
    int n, nq, red[2 * (NT / 64)];
};

// Behind `have` keys, the first k - have entries of key `low` in order of their places; how many keys there are then.  The workgroup goes along the row
// together and stops where it has them.
template <int NT, typename T>
__device__ __forceinline__ int first_ties(const T* x, int n, int first, uint32_t low, int have, int k, TopLds<NT>& s) {
    constexpr int VE = lp_vec<T>::N;
    const int nv = n / VE, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int phase = 0;
    for (int at = 0; have < k && at <= nv; at += NT) {
        const int v = at + (int)threadIdx.x;
        float a[VE];
        if (v < nv) {
            lp_unpack(lp_load16(x + (int64_t)v * VE), a, x);
        } else {
#pragma unroll
            for (int i = 0; i < VE; ++i) a[i] = v == nv && nv * VE + i < n ? lp_float(x[nv * VE + i]) : -INF;
        }
        uint32_t tie = 0;
#pragma unroll
        for (int i = 0; i < VE; ++i) tie |= (a[i] > -INF && key_of(a[i] + 0.f) == low ? 1u : 0u) << i;
        int before = __popc(tie);  // ties of this thread and the lanes before it
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(before, o);
            before += lane >= o ? u : 0;
        }
        int* const r = s.red + (phase ^= 1) * (NT / 64);
        if (lane == 63) r[w] = before;
        __syncthreads();
        int place = have + before - __popc(tie);
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) {
            place += i < w ? r[i] : 0;
            have += r[i];
        }
        for (; tie && place < k; tie &= tie - 1, ++place) s.cand[place] = (uint64_t)low << 32 | (uint32_t)~(first + v * VE + __ffs(tie) - 1);
    }
    return have < k ? have : k;
}

// The k largest keys of the n entries at x, in order, to emit(place, key).  The k-th largest among largest entries of parts of the row bounds the row's
// k-th largest from below, so only about k buckets are read again, as whole lines.  (With one bucket a thread, its vectors NT apart, 100 of 512 buckets
// touched nearly every line of the row: 64 x 1000000, k = 100 took 84 us, 43 without alternatives.)
template <int NT, typename T, typename E>
__device__ __forceinline__ void top_entries(const T* x, int n, int first, int k, int shift, TopLds<NT>& s, E emit) {
    constexpr int VE = lp_vec<T>::N, B = buckets<NT>(), PER = B / NT;
    const int nv = n / VE, all = (nv + (1 << shift) - 1) >> shift, nb = all < B ? all : B;
    int phase = 0;
    if (threadIdx.x == 0) s.n = s.nq = 0;
    __syncthreads();
    uint32_t mine[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {  // a stretch with nothing but -inf and NaN has no key: its largest entry is -inf or, NaN throughout, a NaN
        const float q = i * NT + (int)threadIdx.x < nb ? s.most[i * NT + threadIdx.x] : -INF;
        mine[i] = q > -INF ? key_of(q + 0.f) : 0;
    }
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) largest = mine[i] > largest ? mine[i] : largest;
    // The k-th largest of the threads' largest, from the high bits down to bit `end`: a little below the buckets' own.  One wavefront looks for it, the
    // others' in its registers: no barrier a bit.
    auto bound = [&](int end) {
        uint32_t* const top = reinterpret_cast<uint32_t*>(s.cand);
        top[threadIdx.x] = largest;
        __syncthreads();
        if (threadIdx.x < 64) {
            uint32_t of[NT / 64], t = 0;
#pragma unroll
            for (int w = 0; w < NT / 64; ++w) of[w] = top[w * 64 + threadIdx.x];
            if (nb >= k)
                for (int b = 31; b >= end; --b) {
                    const uint32_t next = t | 1u << b;
                    int c = 0;
#pragma unroll
                    for (int w = 0; w < NT / 64; ++w) c += lanes(of[w] >= next);
                    if (c >= k) t = next;
                }
            if (threadIdx.x == 0) s.low = t;
        }
        __syncthreads();
        return s.low <= KEY_NONE ? KEY_NONE + 1 : s.low;
    };
    uint32_t low = bound(16);
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (mine[i] >= low) s.list[atomicAdd(&s.nq, 1)] = (uint16_t)(i * NT + threadIdx.x);
    __syncthreads();
    const int lap = s.nq << shift, nq = lap * ((all + B - 1) / B);  // vectors to read again: of each round of the buckets
    auto put = [&](uint64_t key) {
        const int at = atomicAdd(&s.n, 1);
        if (at < CAND) s.cand[at] = key;
    };
    for (int p = threadIdx.x; p < nq; p += 4 * NT) {
        uint4 w[4];
        int v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int q = p + j * NT;
            v[j] = q < nq ? ((q / lap * B + s.list[q % lap >> shift]) << shift) + (q & ((1 << shift) - 1)) : nv;
            w[j] = v[j] < nv ? lp_load16(x + (int64_t)v[j] * VE) : all_masked(x);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float a[VE];
            lp_unpack(w[j], a, x);
#pragma unroll
            for (int i = 0; i < VE; ++i)
                if (a[i] > -INF && key_of(a[i] + 0.f) >= low) put(key_at(a[i], first + v[j] * VE + i));
        }
    }
    if (threadIdx.x < n - nv * VE) {
        const float a = lp_float(x[nv * VE + threadIdx.x]);
        if (a > -INF && key_of(a + 0.f) >= low) put(key_at(a, first + nv * VE + threadIdx.x));
    }
    __syncthreads();
    int have = s.n;
    if (__builtin_expect(have > CAND, 0)) {
        // The bound to its last bit (logits of 300 +- 1 are 2 apart in 16 bits), what lies above it, and the first of its ties: a row, or a part of one, of
        // one value, as masks of a finite value leave them, has more than LDS holds (4096 x 131072 bf16 with eleven entries left, 20 alternatives: 585 us; a
        // search of the row for the threshold bit by bit took 8100).
        __syncthreads();
        low = bound(0);
        if (threadIdx.x == 0) s.n = 0;
        __syncthreads();
        each_entry<NT>(x, n, [&](const float(&l)[VE], int at) {
#pragma unroll
            for (int i = 0; i < VE; ++i)
                if (l[i] > -INF && key_of(l[i] + 0.f) > low) put(key_at(l[i], first + at + i));
        });
        __syncthreads();
        have = s.n;
        if (have < k) have = first_ties<NT>(x, n, first, low, have, k, s);
    }
    if (__builtin_expect(have > CAND, 0)) {  // more large entries than that fell to the same few threads: look for the threshold in the row itself
        const uint64_t t = key_threshold(k, CAND, [&](uint64_t next) {
            int c = 0;
            each_entry<NT>(x, n, [&](const float(&l)[VE], int at) {
#pragma unroll
                for (int i = 0; i < VE; ++i) c += key_at(l[i], first + at + i) >= next ? 1 : 0;
            });
#pragma unroll
            for (int o = 32; o; o >>= 1) c += __shfl_xor(c, o);
            return count_block<NT>(c, s.red, phase);
        });
        if (threadIdx.x == 0) s.n = 0;
        __syncthreads();
        each_entry<NT>(x, n, [&](const float(&l)[VE], int at) {
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                const uint64_t key = key_at(l[i], first + at + i);
                if (key && key >= t) put(key);
            }
        });
        __syncthreads();
        have = s.n;
    }
    if (have > NT) {
        const uint64_t t = key_threshold(k, NT, [&](uint64_t next) {
            int c = 0;
            for (int i = 0; i < CAND; i += NT) c += lanes(i + (int)threadIdx.x < have && s.cand[i + threadIdx.x] >= next);
            return count_block<NT>(c, s.red, phase);
        });
        uint64_t keep[CAND / NT];
#pragma unroll
        for (int j = 0; j < CAND / NT; ++j) {
            const int i = threadIdx.x + j * NT;
            keep[j] = i < have ? s.cand[i] : 0;
        }
        __syncthreads();
        if (threadIdx.x == 0) s.n = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < CAND / NT; ++j)
            if (keep[j] && keep[j] >= t) s.cand[atomicAdd(&s.n, 1)] = keep[j];
        __syncthreads();
        have = s.n;
    }
    if (threadIdx.x == 0) s.cand[have] = 0;  // the other of the last pair
    __syncthreads();
    if (threadIdx.x < have) {
        const uint64_t key = s.cand[threadIdx.x];
        const int place = place_of(key, s.cand, have);
        if (place < k) emit(place, key);
    }
    for (int i = have + threadIdx.x; i < k; i += NT) emit(i, (uint64_t)0);
}

// ---- token log probabilities --------------------------------------------------------------------------------------------------------------
struct LpArgs {
    const void* x;
    int64_t ld, N;
    int V, k, parts, chunk;
    const void* ids;
    int ids_dtype;
    float inv_t, c;
    float *logp, *entropy, *lse, *top_logp;
    int32_t* top_ids;
    float* stats;   // [N, 2]: maximum, log2 of the sum
    float4* part;   // [N, parts] sums
    uint64_t* tops;  // [N, parts, k] keys
};

__device__ __forceinline__ int64_t id_at(const void* ids, int dtype, int64_t i) {
    return dtype == MH_I32 ? (int64_t)static_cast<const int32_t*>(ids)[i] : static_cast<const int64_t*>(ids)[i];
}

__device__ __forceinline__ float lp_value(float l, const Sum& t, float inv_t) {
    return t.m == -INF ? -INF : fmaf(l - t.m, inv_t, -logf(t.s));
}

// the row's given id's logit, asked for before the row is read
template <typename T>
__device__ __forceinline__ float lp_given(const LpArgs& g, int64_t row, bool& has) {
    const int64_t id = g.ids ? id_at(g.ids, g.ids_dtype, row) : -1;
    has = id >= 0 && id < g.V;
    return has ? lp_float(static_cast<const T*>(g.x)[row * g.ld + id]) : 0.f;
}
__device__ __forceinline__ void lp_finish(const LpArgs& g, int64_t row, const Sum& t, bool has, float given) {
    const float ls = log2f(t.s);
    const bool none = t.m == -INF;
    if (g.ids) g.logp[row] = has ? lp_value(given, t, g.inv_t) : 0.f;
    g.entropy[row] = none ? 0.f : LN2 * (ls - t.u / t.s);
    g.lse[row] = none ? -INF : fmaf(t.m, g.inv_t, logf(t.s));
    g.stats[2 * row] = t.m;
    g.stats[2 * row + 1] = none ? 0.f : ls;
}

__device__ __forceinline__ void lp_emit(const LpArgs& g, int64_t row, const Sum& t, int place, uint64_t key) {
    g.top_ids[row * g.k + place] = key ? (int32_t)~(uint32_t)key : -1;
    g.top_logp[row * g.k + place] = key ? lp_value(key_value((uint32_t)(key >> 32)), t, g.inv_t) : -INF;
}

// One read of the logits: 8192 x 32769 fp32 (rows at any word) 216 us, 5.0 TB/s; 64 x 1000000 fp32 with 100 alternatives 51 us, 5.0 TB/s;
// 1 x 131072 bf16 with 20 alternatives 9.6 us in parts, the join behind it 7.4: both latency.  Eight wavefronts a SIMD are asked for where the compiler would
// leave room for seven: 4096 x 16384 fp32, 20 alternatives, 52 us and 58.
template <int NT, typename T, bool TOP>
__global__ __launch_bounds__(NT, TOP && NT == 512 ? 8 : 1) void token_logprobs_kernel(const LpArgs g) {
    __shared__ Sum red[NT / 64];
    __shared__ TopLds<TOP ? NT : 64> lds;
    const int64_t row = blockIdx.x / (uint32_t)g.parts;
    const int part = (int)(blockIdx.x % (uint32_t)g.parts), c0 = part * g.chunk, n = g.V - c0 < g.chunk ? g.V - c0 : g.chunk;
    const T* x = static_cast<const T*>(g.x) + row * g.ld + c0;
    float given = 0.f;
    bool has = false;
    if (threadIdx.x == 0 && g.parts == 1) given = lp_given<T>(g, row, has);
    const int shift = n / lp_vec<T>::N <= buckets<NT>() ? 0 : 3;
    const Sum t = read_sums<NT, true, false, TOP>(x, n, g.c, nullptr, TOP ? lds.most : nullptr, shift, red);
    if (threadIdx.x == 0) {
        if (g.parts == 1) lp_finish(g, row, t, has, given);
        else g.part[row * g.parts + part] = make_float4(t.m, t.s, t.u, 0.f);
    }
    if constexpr (TOP) {
        top_entries<NT>(x, n, c0, g.k, shift, lds, [&](int place, uint64_t key) {
            if (g.parts == 1) lp_emit(g, row, t, place, key);
            else g.tops[(row * g.parts + part) * g.k + place] = key;
        });
    }
}

// The sums of a row's parts put together.
template <int NT>
__device__ __forceinline__ Sum join_parts(const float4* part, int parts, float c, Sum* red) {
    Sum a = {-3.402823466e38f, 0.f, 0.f};
    for (int i = threadIdx.x; i < parts; i += NT) {
        const float4 v = part[i];
        if (v.x != -INF) a = sum_join(a, Sum{v.x, v.y, v.z}, c);
    }
    a = sum_block<NT>(a, c, red);
    if (a.s == 0.f) a.m = -INF;
    return a;
}

template <typename T>
__global__ __launch_bounds__(512) void token_logprobs_join_kernel(const LpArgs g) {
    __shared__ __attribute__((aligned(16))) uint64_t cand[512 + 2];
    __shared__ Sum sums[8];
    __shared__ int red[16], have;
    const int64_t row = blockIdx.x;
    const int n = g.parts * g.k;
    const uint64_t* in = g.tops + row * n;
    uint64_t key[JOIN_MOST / 512];
#pragma unroll
    for (int j = 0; j < JOIN_MOST / 512; ++j) key[j] = (int)threadIdx.x + 512 * j < n ? in[threadIdx.x + 512 * j] : 0;
    bool has = false;
    const float given = threadIdx.x == 0 ? lp_given<T>(g, row, has) : 0.f;
    const Sum t = join_parts<512>(g.part + row * g.parts, g.parts, g.c, sums);
    if (threadIdx.x == 0) lp_finish(g, row, t, has, given);
    if (!g.k) return;
    int phase = 0;
    uint64_t th = 1;
    if (n > 512)
        th = key_threshold(g.k, 512, [&](uint64_t next) {
            int c = 0;
#pragma unroll
            for (int j = 0; j < JOIN_MOST / 512; ++j) c += lanes(key[j] >= next);
            return count_block<512>(c, red, phase);
        });
    if (th == 0) th = 1;  // fewer than k keys in all
    if (threadIdx.x == 0) have = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < JOIN_MOST / 512; ++j)
        if (key[j] >= th) cand[atomicAdd(&have, 1)] = key[j];
    __syncthreads();
    if (threadIdx.x == 0) cand[have] = 0;
    __syncthreads();
    if (threadIdx.x < have) {
        const uint64_t mine = cand[threadIdx.x];
        const int place = place_of(mine, cand, have);
        if (place < g.k) lp_emit(g, row, t, place, mine);
    }
    for (int i = have + threadIdx.x; i < g.k; i += 512) lp_emit(g, row, t, i, (uint64_t)0);
}

// ---- gradients -------------------------------------------------------------------------------------------------------------------------------
// d[v] = p (A + B log2 p) with p = 2^((l - m) c - L), then the places that differ: the given id (g added) or the teacher's entries.
struct GradArgs {
    const void* x;
    int64_t ld, N, ldd;
    int V, K, parts, chunk;
    const void* ids;
    int ids_dtype;
    int64_t ld_ids;  // distill_topk
    float inv_t, c;
    const float *stats, *entropy, *dlogp, *dentropy, *dlse;  // token_logprobs: stats [N, 2]
    const float *top_grad, *dloss;                           // distill_topk: stats [N, 3] (maximum, log2 sum, weight)
    void* d;
};

template <typename T, int N>
__device__ __forceinline__ void grad_values(const float (&l)[N], float (&o)[N], float m, float c, float L, float A, float B, bool ent) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float t = fmaf(l[i] - m, c, -L), e = ex2(t);
        o[i] = ent ? e * fmaf(B, fmaxf(t, -200.f), A) : e * A;
    }
}

// A vector at a time: what hides the loads here is the number of wavefronts, and more vectors a thread cost more of those than they bring
// (4096 x 131003 bf16 with entropy: 360 us, 513 with four vectors in flight a thread at 81 registers).
template <int NT, typename T, bool ENT>
__device__ __forceinline__ void grad_row(const T* x, T* d, int n, float m, float c, float L, float A, float B) {
    constexpr int VE = lp_vec<T>::N;
    const int nv = n / VE;
#pragma unroll 1
    for (int v = threadIdx.x; v < nv; v += NT) {
        float l[VE], o[VE];
        lp_unpack(lp_load16(x + (int64_t)v * VE), l, x);
        grad_values<T>(l, o, m, c, L, A, B, ENT);
        lp_store16(d + (int64_t)v * VE, o);
    }
    if (threadIdx.x < n - nv * VE) {
        const int i = nv * VE + threadIdx.x;
        float l[1] = {lp_float(x[i])}, o[1];
        grad_values<T>(l, o, m, c, L, A, B, ENT);
        lp_store(d + i, o[0]);
    }
}
template <int NT, typename T>
__device__ __forceinline__ void zero_row(T* d, int n) {
    constexpr int VE = lp_vec<T>::N;
    float z[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) z[i] = 0.f;
    const int nv = n / VE;
    for (int v = threadIdx.x; v < nv; v += NT) lp_store16(d + (int64_t)v * VE, z);
    if (threadIdx.x < n - nv * VE) lp_store(d + nv * VE + threadIdx.x, 0.f);
}

// 8192 x 32769 fp32 351 us, 6.1 TB/s read and written; 4096 x 131003 bf16 with the entropy's term 347 us, 6.2 TB/s.
template <int NT, typename T>
__global__ __launch_bounds__(NT) void token_logprobs_bwd_kernel(const GradArgs g) {
    const int64_t row = blockIdx.x / (uint32_t)g.parts;
    const int c0 = (int)(blockIdx.x % (uint32_t)g.parts) * g.chunk, n = g.V - c0 < g.chunk ? g.V - c0 : g.chunk;
    const T* x = static_cast<const T*>(g.x) + row * g.ld + c0;
    T* d = static_cast<T*>(g.d) + row * g.ldd + c0;
    const int64_t id = g.ids ? id_at(g.ids, g.ids_dtype, row) : -1;
    const float gr = g.dlogp && id >= 0 && id < g.V ? g.dlogp[row] : 0.f, h = g.dentropy ? g.dentropy[row] : 0.f, z = g.dlse ? g.dlse[row] : 0.f;
    const float m = g.stats[2 * row], L = g.stats[2 * row + 1];
    if (m == -INF || (gr == 0.f && h == 0.f && z == 0.f)) {
        zero_row<NT>(d, n);
        return;
    }
    const float A = (z - gr - h * g.entropy[row]) * g.inv_t, B = -h * LN2 * g.inv_t;
    const bool here = gr != 0.f && id >= c0 && id < c0 + n;
    const float lt = here && threadIdx.x == 0 ? lp_float(x[id - c0]) : 0.f;  // before d, which may be x, is written
    __syncthreads();
    if (h != 0.f) grad_row<NT, T, true>(x, d, n, m, g.c, L, A, B);
    else grad_row<NT, T, false>(x, d, n, m, g.c, L, A, 0.f);
    if (here) {
        __syncthreads();
        if (threadIdx.x == 0) {
            float l[1] = {lt}, o[1];
            grad_values<T>(l, o, m, g.c, L, A, B, h != 0.f);
            lp_store(d + (id - c0), fmaf(gr, g.inv_t, o[0]));
        }
    }
}

// ---- distillation ------------------------------------------------------------------------------------------------------------------------------
// q_k: the teacher's mass on its entries -- softmax of the K log probabilities (tail = 0), or their exponentials, with r = 1 - sum q for the rest of
// the catalogue (tail = 1).  loss = sum q_k (ln q_k - ln p_k) + r (ln r - ln p_rest);  d loss / d z = c p - sum of its q at an entry, c = sum q + r,
// and (c p_rest - r) p / p_rest elsewhere.  With a tail the pass leaves the entries out, by a bit for each column in LDS, so p_rest is a sum of its
// own and not what is left of 1.  The K entries themselves are done in fp64: few, and 1 - sum q cancels.
struct DsArgs {
    const void* x;
    int64_t ld, N;
    int V, K, parts, chunk, tail;
    const void* ids;
    int ids_dtype;
    int64_t ld_ids, ld_tlp;
    const float* tlp;
    float inv_t, c;
    float *loss, *stats, *top_grad;
    float4* part;
};

// One wavefront does a row's entries, E of them a lane (entry lane + 64 i), by shuffles alone.
constexpr int SEEN = 2 * TOP_MOST;
struct DsLds {
    double q[TOP_MOST];
    int id[TOP_MOST], seen[SEEN];
};
template <int E>
struct DsTeacher {
    int id[E];         // -1: none
    bool first[E];     // no entry before has the same id
    float l[E];        // the student's logit
    double q[E], lq[E];  // the teacher's mass, and its logarithm
    double of_id[E];   // all entries' mass on this id
    double Q;          // the entries' mass
    bool any;          // the row has a teacher
};
// LDS written before is read after, by the same wavefront
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <int E, typename T>
__device__ __forceinline__ void ds_teacher(const DsArgs& g, int64_t row, DsLds& s, DsTeacher<E>& e) {
    const int lane = threadIdx.x & 63;
    float tl[E], tm = -INF;
    bool some = false;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int j = lane + 64 * i;
        e.id[i] = -1, tl[i] = -INF;
        if (j < g.K) {
            const int64_t v = id_at(g.ids, g.ids_dtype, row * g.ld_ids + j);
            if (v >= 0 && v < g.V) e.id[i] = (int)v, tl[i] = g.tlp[row * g.ld_tlp + j];
        }
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
        e.l[i] = e.id[i] >= 0 ? lp_float(static_cast<const T*>(g.x)[row * g.ld + e.id[i]]) : -INF;
        tm = fmaxf(tm, tl[i]);
        some |= e.id[i] >= 0 && (g.tail || !(tl[i] == -INF));  // NaN counts: it has to show
    }
    e.any = __any(some);
    tm = g.tail ? 0.f : max_wave(tm);
    e.Q = 0.0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        e.lq[i] = e.any ? (double)tl[i] - tm : 0.0;
        e.q[i] = e.id[i] >= 0 && e.any ? exp(e.lq[i]) : 0.0;
        e.Q += e.q[i];
    }
    e.Q = add_wave(e.Q);
    if (!g.tail && e.any) {
        const double lQ = log(e.Q);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            e.q[i] /= e.Q;
            e.lq[i] -= lQ;
        }
        e.Q = 1.0;
    }
    // Does the row give an id twice?  A table of twice as many places as entries tells; only then are the entries compared with each other.
    for (int i = lane; i < SEEN; i += 64) s.seen[i] = -1;
    wave_fence();
    bool twice = false;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        e.first[i] = e.id[i] >= 0;
        e.of_id[i] = e.q[i];
        if (e.id[i] >= 0) {
            uint32_t h = ((uint32_t)e.id[i] * 2654435761u) / (0x80000000u / (SEEN / 2));
            for (int was; (was = atomicCAS(&s.seen[h], -1, e.id[i])) != -1; h = (h + 1) & (SEEN - 1))
                if (was == e.id[i]) {
                    twice = true;
                    break;
                }
        }
    }
    if (__any(twice)) {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (lane + 64 * i < g.K) s.id[lane + 64 * i] = e.id[i], s.q[lane + 64 * i] = e.q[i];
        wave_fence();
#pragma unroll
        for (int i = 0; i < E; ++i) e.of_id[i] = 0.0;
#pragma unroll 4
        for (int j = 0; j < g.K; ++j) {
            const int id = s.id[j];
            const double q = s.q[j];
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const bool same = id == e.id[i];
                e.of_id[i] += same ? q : 0.0;
                if (same && j < lane + 64 * i) e.first[i] = false;
            }
        }
    }
}

// The row's loss, the entries' gradients and the weight of the other columns, from t: the sums over the row (tail: over the row without the
// teacher's entries).
template <int E>
__device__ __forceinline__ float ds_loss(const DsArgs& g, const Sum& t, const DsTeacher<E>& e, float& loss, float (&grad)[E]) {
    float m = t.m;
    double sum = t.s;
    if (g.tail) {
        float lm = -INF;
#pragma unroll
        for (int i = 0; i < E; ++i) lm = fmaxf(lm, e.l[i]);
        m = fmaxf(m, max_wave(lm));
        sum = 0.0;
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (e.first[i] && !(e.l[i] == -INF)) sum += exp((double)(e.l[i] - m) * g.inv_t);
        sum = add_wave(sum) + (t.m == -INF ? 0.0 : (double)t.s * exp((double)(t.m - m) * g.inv_t));
    }
    const double ln_s = log(sum);
    const bool none = m == -INF;  // the student's row is masked throughout
    double lp[E], total = 0.0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        lp[i] = none ? -(double)INF : (double)(e.l[i] - m) * g.inv_t - ln_s;
        if (e.q[i] > 0.0 || e.q[i] != e.q[i]) total += e.q[i] * (e.lq[i] - lp[i]);
    }
    total = add_wave(total);
    const bool others = g.tail && !(t.m == -INF) && t.s != 0.f;
    const double left = others && e.any && e.Q < 1.0 ? 1.0 - e.Q : 0.0, c = e.Q + left;
    const double lpr = others ? (double)(t.m - m) * g.inv_t + log((double)t.s) - ln_s : 0.0;
    if (left > 0.0) total += left * (log(left) - lpr);
    loss = e.any ? (float)total : 0.f;
    const bool live = e.any && !none;
#pragma unroll
    for (int i = 0; i < E; ++i) grad[i] = live && e.id[i] >= 0 ? (float)(c * exp(lp[i]) - e.of_id[i]) : 0.f;
    if (!live) return 0.f;
    if (!g.tail) return 1.f;
    return others ? (float)(c * exp(lpr) - left) : 0.f;
}

template <int E>
__device__ __forceinline__ void ds_store(const DsArgs& g, int64_t row, const Sum& t, const DsTeacher<E>& e) {
    const int lane = threadIdx.x & 63;
    float loss, grad[E];
    const float w = ds_loss<E>(g, t, e, loss, grad);
    if (lane == 0) g.loss[row] = loss;
    if (g.stats) {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (lane + 64 * i < g.K) g.top_grad[row * g.K + lane + 64 * i] = grad[i];
        if (lane == 0) {
            g.stats[3 * row] = t.m;
            g.stats[3 * row + 1] = t.s > 0.f || t.s != t.s ? log2f(t.s) : 0.f;
            g.stats[3 * row + 2] = w;
        }
    }
}

// A row's parts joined, and its loss: a wavefront a row.
template <int E, typename T>
__global__ __launch_bounds__(256) void distill_topk_finish_kernel(const DsArgs g) {
    __shared__ DsLds lds[4];
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= g.N) return;
    const float4* part = g.part + row * g.parts;
    Sum t = {-3.402823466e38f, 0.f, 0.f};
    for (int i = lane; i < g.parts; i += 64) {
        const float4 v = part[i];
        if (v.x != -INF) t = sum_join(t, Sum{v.x, v.y, v.z}, g.c);
    }
    DsTeacher<E> e;
    ds_teacher<E, T>(g, row, lds[threadIdx.x >> 6], e);
    t = sum_wave(t, g.c);
    if (t.s == 0.f) t.m = -INF;
    ds_store<E>(g, row, t, e);
}

// bit i of `bits`: column c0 + i is one of the row's teacher entries
__device__ __forceinline__ void ds_bits(const DsArgs& g, int64_t row, int c0, int n, uint32_t* bits) {
    for (int i = threadIdx.x; i < (n + 31) / 32; i += blockDim.x) bits[i] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < g.K; j += blockDim.x) {
        const int64_t v = id_at(g.ids, g.ids_dtype, row * g.ld_ids + j);
        if (v >= c0 && v < c0 + n) atomicOr(&bits[(v - c0) >> 5], 1u << ((v - c0) & 31));
    }
    __syncthreads();
}

// The sums of a row, or a part of one, with a tail without the teacher's entries.  E != 0: a row a workgroup, which has one wavefront more for the
// teacher's entries, done while the others read.  2048 x 50021 f16, 64 entries: 36 us, 5.6 TB/s; 4096 x 131072 bf16, 128 entries and a tail: 233 us
// (200 at best), 4.6 TB/s.
template <int NT, int E, typename T, bool TAIL>
__global__ __launch_bounds__(NT + (E ? 64 : 0), E == 1 || E == 2 ? 8 : 1) void distill_topk_sums_kernel(const DsArgs g) {
    extern __shared__ uint32_t bits[];
    __shared__ Sum red[NT / 64];
    const int64_t row = E ? blockIdx.x : blockIdx.x / (uint32_t)g.parts;
    const int part = E ? 0 : (int)(blockIdx.x % (uint32_t)g.parts), c0 = part * g.chunk, n = g.V - c0 < g.chunk ? g.V - c0 : g.chunk;
    if (TAIL) ds_bits(g, row, c0, n, bits);
    const T* x = static_cast<const T*>(g.x) + row * g.ld + c0;
    if constexpr (E != 0) {
        __shared__ DsLds lds;
        DsTeacher<E> e;
        if (threadIdx.x >= NT) ds_teacher<E, T>(g, row, lds, e);
        const Sum t = read_sums<NT, false, TAIL, false>(x, n, g.c, bits, nullptr, 0, red);
        if (threadIdx.x >= NT) ds_store<E>(g, row, t, e);
    } else {
        const Sum t = read_sums<NT, false, TAIL, false>(x, n, g.c, bits, nullptr, 0, red);
        if (threadIdx.x == 0) g.part[row * g.parts + part] = make_float4(t.m, t.s, t.u, 0.f);
    }
}

// 4096 x 131072 bf16, 128 entries: 327 us, 6.6 TB/s read and written.
template <int NT, typename T>
__global__ __launch_bounds__(NT) void distill_topk_bwd_kernel(const GradArgs g) {
    const int64_t row = blockIdx.x / (uint32_t)g.parts;
    const int c0 = (int)(blockIdx.x % (uint32_t)g.parts) * g.chunk, n = g.V - c0 < g.chunk ? g.V - c0 : g.chunk;
    const T* x = static_cast<const T*>(g.x) + row * g.ld + c0;
    T* d = static_cast<T*>(g.d) + row * g.ldd + c0;
    const float f = (g.dloss ? g.dloss[row] : 1.f) * g.inv_t, A = g.stats[3 * row + 2] * f;
    if (A == 0.f) zero_row<NT>(d, n);
    else grad_row<NT, T, false>(x, d, n, g.stats[3 * row], g.c, g.stats[3 * row + 1], A, 0.f);
    __syncthreads();
    for (int j = threadIdx.x; j < g.K; j += NT) {
        const int64_t v = id_at(g.ids, g.ids_dtype, row * g.ld_ids + j);
        if (v >= c0 && v < c0 + n) lp_store(d + (v - c0), f == 0.f ? 0.f : g.top_grad[row * g.K + j] * f);  // an id given twice has one value
    }
}

// A row's loss and gradient from one read: the row stays in registers, R 16-byte vectors a thread, between its sums and its gradient.
// Hides from the compiler that a vector is what it was: it would unpack the whole row beforehand and keep the values of one use for the next, at two to
// four times the registers.
__device__ __forceinline__ void forget(uint4& w) { asm volatile("" : "+v"(w.x), "+v"(w.y), "+v"(w.z), "+v"(w.w)); }

// p, the same for all threads, and a thread's offset in bytes: one address register instead of two for every access
template <typename T>
__device__ __forceinline__ T* at_offset(T* p, uint32_t bytes) {
    typedef typename std::conditional<std::is_const<T>::value, const char, char>::type byte;
    return reinterpret_cast<T*>(reinterpret_cast<byte*>(p) + bytes);
}

template <int NT, int R, int E, typename T, bool TAIL>
__global__ __launch_bounds__(NT) void distill_topk_train_kernel(const DsArgs g, const float* dloss, T* dall, int64_t ldd) {  // dall may be g.x
    constexpr int VE = lp_vec<T>::N;
    extern __shared__ uint32_t bits[];
    __shared__ Sum red[NT / 64];
    __shared__ DsLds lds;
    __shared__ float weight;
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(g.x) + row * g.ld;
    T* d = dall + row * ldd;
    const int nv = g.V / VE, rest = g.V - nv * VE;
    const float f = (dloss ? dloss[row] : 1.f) * g.inv_t;
    uint4 w[R];
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const int v = threadIdx.x + j * NT;
        w[j] = v < nv ? lp_load16(at_offset(x + j * NT * VE, threadIdx.x * 16)) : all_masked(x);
    }
    const int last = nv * VE + threadIdx.x;  // this thread's entry behind the vectors
    const float one = threadIdx.x < rest ? lp_float(x[last]) : -INF;
    if (TAIL) ds_bits(g, row, 0, g.V, bits);
    DsTeacher<E> e;
    if (threadIdx.x < 64) ds_teacher<E, T>(g, row, lds, e);  // the first wavefront, while the others add
    auto values = [&](int j, float (&a)[VE]) {
        forget(w[j]);
        lp_unpack(w[j], a, x);
        if (TAIL) {
            const int v = threadIdx.x + j * NT;
            if (v < nv) mask_values(a, bits, v);
        }
    };
    const bool skip_one = TAIL && threadIdx.x < rest && (bits[last >> 5] >> (last & 31) & 1);
    Run run(g.c);
    float most = -INF;
#pragma unroll
    for (int j = 0; j < R; ++j) {
        float a[VE];
        values(j, a);
        const float b = most_of(a);
        most = fmaxf(most, b);
        run.template take<false>(a, b, g.c);
        asm volatile("" : "+v"(run.s));  // added up here, not behind the barrier that follows: one vector's values live at a time
    }
    {
        const float a[1] = {skip_one ? -INF : one};
        most = fmaxf(most, a[0]);
        run.template take<false>(a, a[0], g.c);
    }
    const bool beyond = __syncthreads_or(!(run.B < 2.f * FAR));
    Sum t = sum_block<NT>(run.sum(g.c), g.c, red);
    if (t.s < 0.5f || beyond) {  // as in read_sums
        t = Sum{max_block<NT>(most, reinterpret_cast<float*>(red)), 0.f, 0.f};
        if (t.m != -INF) {
            Sum a = {t.m, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < R; ++j) {
                float l[VE];
                values(j, l);
#pragma unroll
                for (int i = 0; i < VE; ++i) a.s += ex2((l[i] - t.m) * g.c);
                asm volatile("" : "+v"(a.s));
            }
            a.s += ex2(((skip_one ? -INF : one) - t.m) * g.c);
            t = sum_block<NT>(a, g.c, red);
        }
    }
    float loss, grad[E];
    if (threadIdx.x < 64) {
        const float wt = ds_loss<E>(g, t, e, loss, grad);
        if (threadIdx.x == 0) {
            g.loss[row] = loss;
            weight = wt;
        }
    }
    __syncthreads();
    const float A = weight * f;
    if (A == 0.f) {
        zero_row<NT>(d, g.V);
    } else {
        const float L = log2f(t.s);
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const int v = threadIdx.x + j * NT;
            if (v < nv) {
                float l[VE], o[VE];
                forget(w[j]);
                lp_unpack(w[j], l, x);
                grad_values<T>(l, o, t.m, g.c, L, A, 0.f, false);
                lp_store16(at_offset(d + j * NT * VE, threadIdx.x * 16), o);
            }
        }
        if (threadIdx.x < rest) {
            const float l[1] = {one};
            float o[1];
            grad_values<T>(l, o, t.m, g.c, L, A, 0.f, false);
            lp_store(d + last, o[0]);
        }
    }
    __syncthreads();
    if (threadIdx.x < 64) {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (e.id[i] >= 0) lp_store(d + e.id[i], f == 0.f ? 0.f : grad[i] * f);
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------------------------
// Parts of a row: one, unless the rows alone do not fill the chip.
void plan_parts(int64_t N, int64_t V, int64_t most, int64_t least, int& parts, int& chunk) {
    int64_t p = mh_ceil_div(1024, N);
    if (p > mh_ceil_div(V, 8192)) p = mh_ceil_div(V, 8192);
    if (p > most) p = most;
    if (p < least) p = least;
    const int64_t c = mh_ceil_div(mh_ceil_div(V, p), 64) * 64;
    chunk = (int)c;
    parts = (int)mh_ceil_div(V, c);
}
void lp_plan(int64_t N, int64_t V, int k, int& parts, int& chunk) { plan_parts(N, V, k ? JOIN_MOST / k : 1024, 1, parts, chunk); }
void ds_plan(int64_t N, int64_t V, bool tail, int& parts, int& chunk) { plan_parts(N, V, 1024, tail ? mh_ceil_div(V, TAIL_CHUNK - 64) : 1, parts, chunk); }

int32_t ts_check(const char* who, const void* x, int32_t dtype, int64_t ld, int64_t N, int64_t V, int32_t ids_dtype, float T) {
    MH_REQUIRE(N >= 0 && V >= 1 && V < ((int64_t)1 << 31) - 65536 && N < (int64_t)1 << 31 && ld >= V, "%s: sizes N=%lld V=%lld ld=%lld", who, (long long)N,
               (long long)V, (long long)ld);
    MH_REQUIRE(dtype == MH_F32 || dtype == MH_BF16 || dtype == MH_F16, "%s: unknown type %d", who, (int)dtype);
    MH_REQUIRE(ids_dtype == MH_I32 || ids_dtype == MH_I64, "%s: ids must be int32 or int64", who);
    MH_REQUIRE(T >= 1e-4f && T <= 1e4f, "%s: temperature %g is outside [1e-4, 1e4]", who, (double)T);
    MH_REQUIRE(N == 0 || x, "%s: logits is NULL", who);
    return MH_OK;
}
// a gradient lies in place of the logits or apart from them
int32_t ts_gradient(const char* who, const void* x, int32_t dtype, int64_t ld, const void* d, int64_t ldd, int64_t N, int64_t V) {
    const int64_t es = dtype == MH_F32 ? 4 : 2;
    MH_REQUIRE(d != x || ldd == ld, "%s: a gradient in place of the logits needs their leading dimension", who);
    MH_REQUIRE(d == x || !lp_shared(x, ld * es, V * es, N, d, ldd * es, V * es, N), "%s: the gradient overlaps the logits and does not lie in their place", who);
    return MH_OK;
}
// a launch has fewer than 2^32 threads
int32_t ts_grid(const char* who, int64_t N, int parts) {
    MH_REQUIRE(N * parts < (int64_t)1 << 23, "%s: %lld rows in %d parts each are too many workgroups for one call", who, (long long)N, parts);
    return MH_OK;
}
int32_t ts_workspace(const char* who, const void* ws, int64_t bytes, int64_t need) {
    if (need > 0 && (!ws || bytes < need || (reinterpret_cast<uintptr_t>(ws) & 15))) {
        mh_set_error("%s: workspace too small or not 16-byte aligned (%lld bytes, %lld needed)", who, (long long)bytes, (long long)need);
        return MH_ERR_WORKSPACE;
    }
    return MH_OK;
}

// threads of a row's (or part's) workgroup
constexpr int64_t SHORT_ROW = 4096;
// What a workgroup of a gradient (512 threads) reads, and writes as much: workgroups start in order, so short ones keep the chip's accesses in one stretch
// of memory, and the lines a workgroup wrote are still in L2 when the teacher's entries are put in; shorter than two vectors a thread, starting them
// is what takes the time.  4096 x 131072 in bf16: distillation with 128 entries 399 / 353 / 373 / 404 us at 8 / 16 / 24 / 32 KB (442 with a workgroup
// a row), log probabilities and entropy 465 / 372 / 355 / 368 (one box, side by side).
constexpr int64_t GRAD_BYTES_LOGPROBS = 24576, GRAD_BYTES_DISTILL = 16384;

template <typename T>
void lp_launch(const LpArgs& g, hipStream_t s) {
    const dim3 grid((unsigned)(g.N * g.parts));
    if (g.chunk <= SHORT_ROW) {
        if (g.k) MH_LAUNCH((token_logprobs_kernel<256, T, true>), grid, dim3(256), 0, s, g);
        else MH_LAUNCH((token_logprobs_kernel<256, T, false>), grid, dim3(256), 0, s, g);
    } else {
        if (g.k) MH_LAUNCH((token_logprobs_kernel<512, T, true>), grid, dim3(512), 0, s, g);
        else MH_LAUNCH((token_logprobs_kernel<512, T, false>), grid, dim3(512), 0, s, g);
    }
    if (g.parts > 1) MH_LAUNCH(token_logprobs_join_kernel<T>, dim3((unsigned)g.N), dim3(512), 0, s, g);
}
template <int E, typename T>
void ds_launch_sums(const DsArgs& g, hipStream_t s) {
    const dim3 grid((unsigned)(g.N * g.parts));
    const size_t lds = g.tail ? (size_t)(g.chunk + 31) / 32 * 4 : 0;
    constexpr int NT = E ? 448 : 512;  // eight wavefronts in all: four workgroups fill a compute unit
    if (g.chunk <= SHORT_ROW) {
        if (g.tail) MH_LAUNCH((distill_topk_sums_kernel<256, E, T, true>), grid, dim3(256 + (E ? 64 : 0)), lds, s, g);
        else MH_LAUNCH((distill_topk_sums_kernel<256, E, T, false>), grid, dim3(256 + (E ? 64 : 0)), lds, s, g);
    } else {
        if (g.tail) MH_LAUNCH((distill_topk_sums_kernel<NT, E, T, true>), grid, dim3(512), lds, s, g);
        else MH_LAUNCH((distill_topk_sums_kernel<NT, E, T, false>), grid, dim3(512), lds, s, g);
    }
}
template <typename T>
void ds_launch(const DsArgs& g, hipStream_t s) {
    if (g.parts == 1) {
        if (g.K <= 64) ds_launch_sums<1, T>(g, s);
        else if (g.K <= 128) ds_launch_sums<2, T>(g, s);
        else ds_launch_sums<4, T>(g, s);
        return;
    }
    ds_launch_sums<0, T>(g, s);
    const dim3 rows((unsigned)mh_ceil_div(g.N, 4));
    if (g.K <= 64) MH_LAUNCH((distill_topk_finish_kernel<1, T>), rows, dim3(256), 0, s, g);
    else if (g.K <= 128) MH_LAUNCH((distill_topk_finish_kernel<2, T>), rows, dim3(256), 0, s, g);
    else MH_LAUNCH((distill_topk_finish_kernel<4, T>), rows, dim3(256), 0, s, g);
}
// Whether loss and gradient are one launch and one read: the row has to stay in registers, and the one wavefront that does the teacher's entries must
// not be what the workgroup waits for, unless the rows are few and the launches are what counts.  In bf16, one launch against three: 16 x 1009, 5
// entries 14 / 20 us; 2048 x 32768, 64 entries 68 / 79; 8192 x 32768, 64 entries 278 / 320; 256 entries: 512 rows 45 / 60, 2048 rows 155 / 123.
template <typename T>
bool ds_train_once(int64_t N, int64_t V, int K) {
    return V <= 512 * 8 * lp_vec<T>::N && (K <= 64 || N <= 1024);
}
template <int E, typename T>
void ds_train_launch(const DsArgs& g, const float* dloss, T* out, int64_t ldd, hipStream_t s) {
    constexpr int VE = lp_vec<T>::N;
    const dim3 grid((unsigned)g.N);
    const size_t lds = g.tail ? (size_t)(g.V + 31) / 32 * 4 : 0;
#define DS_TRAIN(NT, R)                                                                                                           \
    do {                                                                                                                          \
        if (g.tail) MH_LAUNCH((distill_topk_train_kernel<NT, R, E, T, true>), grid, dim3(NT), lds, s, g, dloss, out, ldd);         \
        else MH_LAUNCH((distill_topk_train_kernel<NT, R, E, T, false>), grid, dim3(NT), lds, s, g, dloss, out, ldd);               \
    } while (0)
    if (g.V <= 256 * 2 * VE) DS_TRAIN(256, 2);
    else if (g.V <= 512 * 4 * VE) DS_TRAIN(512, 4);
    else DS_TRAIN(512, 8);
#undef DS_TRAIN
}
template <typename T>
void ds_train(const DsArgs& g, const float* dloss, void* d, int64_t ldd, hipStream_t s) {
    T* out = static_cast<T*>(d);
    if (g.K <= 64) ds_train_launch<1, T>(g, dloss, out, ldd, s);
    else if (g.K <= 128) ds_train_launch<2, T>(g, dloss, out, ldd, s);
    else ds_train_launch<4, T>(g, dloss, out, ldd, s);
}
template <typename T>
int32_t grad_launch(const char* who, GradArgs g, bool distill, hipStream_t s) {
    plan_parts(g.N, g.V, 1 << 20, mh_ceil_div(g.V * (int64_t)sizeof(T), distill ? GRAD_BYTES_DISTILL : GRAD_BYTES_LOGPROBS), g.parts, g.chunk);
    if (int32_t rc = ts_grid(who, g.N, g.parts)) return rc;
    const dim3 grid((unsigned)(g.N * g.parts));
    if (distill) MH_LAUNCH((distill_topk_bwd_kernel<512, T>), grid, dim3(512), 0, s, g);
    else MH_LAUNCH((token_logprobs_bwd_kernel<512, T>), grid, dim3(512), 0, s, g);
    MH_CHECK_LAUNCH(who);
    return MH_OK;
}
int32_t grad_any(const char* who, const GradArgs& g, int32_t dtype, bool distill, hipStream_t s) {
    if (int32_t rc = ts_gradient(who, g.x, dtype, g.ld, g.d, g.ldd, g.N, g.V)) return rc;
    if (dtype == MH_F32) return grad_launch<float>(who, g, distill, s);
    if (dtype == MH_BF16) return grad_launch<lp_bf16>(who, g, distill, s);
    return grad_launch<lp_f16>(who, g, distill, s);
}

}  // namespace

extern "C" {

int64_t mh_token_logprobs_workspace_bytes(int64_t N, int64_t V, int32_t k) {
    if (N <= 0 || V <= 0 || V >= (int64_t)1 << 31 || k < 0 || k > TOP_MOST) return 0;
    int parts, chunk;
    lp_plan(N, V, k, parts, chunk);
    return parts == 1 ? 0 : N * parts * (16 + 8 * (int64_t)k);
}

int32_t mh_token_logprobs(const void* logits, int32_t dtype, int64_t ld, int64_t N, int64_t V, const void* ids, int32_t ids_dtype, int32_t k,
                          float temperature, float* logp, float* entropy, float* lse, float* top_logp, int32_t* top_ids, float* stats, void* workspace,
                          int64_t workspace_bytes, mh_stream_t stream) {
    if (int32_t rc = ts_check("mh_token_logprobs", logits, dtype, ld, N, V, ids_dtype, temperature)) return rc;
    MH_REQUIRE(k >= 0 && k <= TOP_MOST && k <= V, "mh_token_logprobs: %d alternatives of %lld entries (at most %d)", (int)k, (long long)V, TOP_MOST);
    if (N == 0) return MH_OK;
    MH_REQUIRE(entropy && lse && stats && (!ids || logp) && (k == 0 || (top_logp && top_ids)), "mh_token_logprobs: an output is NULL");
    LpArgs g = {};
    g.x = logits, g.ld = ld, g.N = N, g.V = (int)V, g.k = k, g.ids = ids, g.ids_dtype = ids_dtype;
    g.inv_t = 1.f / temperature, g.c = (float)(1.4426950408889634074 / (double)temperature);
    g.logp = logp, g.entropy = entropy, g.lse = lse, g.top_logp = top_logp, g.top_ids = top_ids, g.stats = stats;
    lp_plan(N, V, k, g.parts, g.chunk);
    if (int32_t rc = ts_grid("mh_token_logprobs", N, g.parts)) return rc;
    if (int32_t rc = ts_workspace("mh_token_logprobs", workspace, workspace_bytes, mh_token_logprobs_workspace_bytes(N, V, k))) return rc;
    g.part = static_cast<float4*>(workspace);
    g.tops = reinterpret_cast<uint64_t*>(g.part + N * g.parts);
    hipStream_t s = mh_stream(stream);
    if (dtype == MH_F32) lp_launch<float>(g, s);
    else if (dtype == MH_BF16) lp_launch<lp_bf16>(g, s);
    else lp_launch<lp_f16>(g, s);
    MH_CHECK_LAUNCH("mh_token_logprobs");
    return MH_OK;
}

int32_t mh_token_logprobs_bwd(const void* logits, int32_t dtype, int64_t ld, int64_t N, int64_t V, const void* ids, int32_t ids_dtype, float temperature,
                              const float* stats, const float* entropy, const float* dlogp, const float* dentropy, const float* dlse, void* dlogits,
                              int64_t ldd, mh_stream_t stream) {
    if (int32_t rc = ts_check("mh_token_logprobs_bwd", logits, dtype, ld, N, V, ids_dtype, temperature)) return rc;
    if (N == 0) return MH_OK;
    MH_REQUIRE(stats && dlogits && ldd >= V && (!dentropy || entropy) && (!dlogp || ids), "mh_token_logprobs_bwd: an argument is NULL, or rows of %lld entries",
               (long long)ldd);
    GradArgs g = {};
    g.x = logits, g.ld = ld, g.N = N, g.ldd = ldd, g.V = (int)V, g.ids = ids, g.ids_dtype = ids_dtype;
    g.inv_t = 1.f / temperature, g.c = (float)(1.4426950408889634074 / (double)temperature);
    g.stats = stats, g.entropy = entropy, g.dlogp = dlogp, g.dentropy = dentropy, g.dlse = dlse, g.d = dlogits;
    return grad_any("mh_token_logprobs_bwd", g, dtype, false, mh_stream(stream));
}

int64_t mh_distill_topk_workspace_bytes(int64_t N, int64_t V, int32_t tail) {
    if (N <= 0 || V <= 0 || V >= (int64_t)1 << 31) return 0;
    int parts, chunk;
    ds_plan(N, V, tail != 0, parts, chunk);
    return parts == 1 ? 0 : N * parts * 16;
}

int32_t mh_distill_topk(const void* logits, int32_t dtype, int64_t ld, int64_t N, int64_t V, const void* teacher_ids, int32_t ids_dtype,
                        int64_t ld_ids, const float* teacher_logp, int64_t ld_logp, int32_t K, float temperature, int32_t tail, float* loss, float* stats,
                        float* top_grad, void* workspace, int64_t workspace_bytes, mh_stream_t stream) {
    if (int32_t rc = ts_check("mh_distill_topk", logits, dtype, ld, N, V, ids_dtype, temperature)) return rc;
    MH_REQUIRE(K >= 1 && K <= TOP_MOST, "mh_distill_topk: %d teacher entries a row (1 to %d)", (int)K, TOP_MOST);
    if (N == 0) return MH_OK;
    MH_REQUIRE(teacher_ids && teacher_logp && loss && (!stats == !top_grad) && ld_ids >= K && ld_logp >= K,
               "mh_distill_topk: an argument is NULL, or the teacher's rows are shorter than %d", (int)K);
    DsArgs g = {};
    g.x = logits, g.ld = ld, g.N = N, g.V = (int)V, g.K = K, g.tail = tail != 0, g.ids = teacher_ids, g.ids_dtype = ids_dtype, g.tlp = teacher_logp, g.ld_ids = ld_ids, g.ld_tlp = ld_logp;
    g.inv_t = 1.f / temperature, g.c = (float)(1.4426950408889634074 / (double)temperature);
    g.loss = loss, g.stats = stats, g.top_grad = top_grad;
    ds_plan(N, V, tail != 0, g.parts, g.chunk);
    if (int32_t rc = ts_grid("mh_distill_topk", N, g.parts)) return rc;
    if (int32_t rc = ts_workspace("mh_distill_topk", workspace, workspace_bytes, mh_distill_topk_workspace_bytes(N, V, tail))) return rc;
    g.part = static_cast<float4*>(workspace);
    hipStream_t s = mh_stream(stream);
    if (dtype == MH_F32) ds_launch<float>(g, s);
    else if (dtype == MH_BF16) ds_launch<lp_bf16>(g, s);
    else ds_launch<lp_f16>(g, s);
    MH_CHECK_LAUNCH("mh_distill_topk");
    return MH_OK;
}

int64_t mh_distill_topk_train_workspace_bytes(int64_t N, int64_t V, int32_t K, int32_t dtype, int32_t tail) {
    if (N <= 0 || V <= 0 || V >= (int64_t)1 << 31 || K < 1 || K > TOP_MOST) return 0;
    if (dtype == MH_F32 ? ds_train_once<float>(N, V, K) : ds_train_once<lp_bf16>(N, V, K)) return 0;
    return mh_distill_topk_workspace_bytes(N, V, tail) + N * (3 + (int64_t)K) * 4;
}

int32_t mh_distill_topk_train(const void* logits, int32_t dtype, int64_t ld, int64_t N, int64_t V, const void* teacher_ids, int32_t ids_dtype, int64_t ld_ids,
                              const float* teacher_logp, int64_t ld_logp, int32_t K, float temperature, int32_t tail, const float* dloss, float* loss,
                              void* dlogits, int64_t ldd, void* workspace, int64_t workspace_bytes, mh_stream_t stream) {
    if (int32_t rc = ts_check("mh_distill_topk_train", logits, dtype, ld, N, V, ids_dtype, temperature)) return rc;
    MH_REQUIRE(K >= 1 && K <= TOP_MOST, "mh_distill_topk_train: %d teacher entries a row (1 to %d)", (int)K, TOP_MOST);
    if (N == 0) return MH_OK;
    MH_REQUIRE(teacher_ids && teacher_logp && loss && dlogits && ld_ids >= K && ld_logp >= K && ldd >= V,
               "mh_distill_topk_train: an argument is NULL, or rows are too short");
    if (int32_t rc = ts_gradient("mh_distill_topk_train", logits, dtype, ld, dlogits, ldd, N, V)) return rc;
    if (int32_t rc = ts_grid("mh_distill_topk_train", N, 1)) return rc;
    const int64_t need = mh_distill_topk_train_workspace_bytes(N, V, K, dtype, tail);
    if (int32_t rc = ts_workspace("mh_distill_topk_train", workspace, workspace_bytes, need)) return rc;
    if (need) {
        char* ws = static_cast<char*>(workspace);
        const int64_t parts = mh_distill_topk_workspace_bytes(N, V, tail);
        float *stats = reinterpret_cast<float*>(ws + parts), *top_grad = stats + 3 * N;
        if (int32_t rc = mh_distill_topk(logits, dtype, ld, N, V, teacher_ids, ids_dtype, ld_ids, teacher_logp, ld_logp, K, temperature, tail, loss, stats,
                                         top_grad, ws, parts, stream))
            return rc;
        return mh_distill_topk_bwd(logits, dtype, ld, N, V, teacher_ids, ids_dtype, ld_ids, K, temperature, stats, top_grad, dloss, dlogits, ldd, stream);
    }
    DsArgs g = {};
    g.x = logits, g.ld = ld, g.N = N, g.V = (int)V, g.K = K, g.tail = tail != 0, g.ids = teacher_ids, g.ids_dtype = ids_dtype, g.ld_ids = ld_ids;
    g.tlp = teacher_logp, g.ld_tlp = ld_logp, g.inv_t = 1.f / temperature, g.c = (float)(1.4426950408889634074 / (double)temperature);
    g.loss = loss;
    hipStream_t s = mh_stream(stream);
    if (dtype == MH_F32) ds_train<float>(g, dloss, dlogits, ldd, s);
    else if (dtype == MH_BF16) ds_train<lp_bf16>(g, dloss, dlogits, ldd, s);
    else ds_train<lp_f16>(g, dloss, dlogits, ldd, s);
    MH_CHECK_LAUNCH("mh_distill_topk_train");
    return MH_OK;
}

int32_t mh_distill_topk_bwd(const void* logits, int32_t dtype, int64_t ld, int64_t N, int64_t V, const void* teacher_ids, int32_t ids_dtype, int64_t ld_ids, int32_t K,
                            float temperature, const float* stats, const float* top_grad, const float* dloss, void* dlogits, int64_t ldd,
                            mh_stream_t stream) {
    if (int32_t rc = ts_check("mh_distill_topk_bwd", logits, dtype, ld, N, V, ids_dtype, temperature)) return rc;
    MH_REQUIRE(K >= 1 && K <= TOP_MOST, "mh_distill_topk_bwd: %d teacher entries a row (1 to %d)", (int)K, TOP_MOST);
    if (N == 0) return MH_OK;
    MH_REQUIRE(teacher_ids && stats && top_grad && dlogits && ldd >= V && ld_ids >= K, "mh_distill_topk_bwd: an argument is NULL, or rows of %lld entries",
               (long long)ldd);
    GradArgs g = {};
    g.x = logits, g.ld = ld, g.N = N, g.ldd = ldd, g.V = (int)V, g.K = K, g.ids = teacher_ids, g.ids_dtype = ids_dtype, g.ld_ids = ld_ids;
    g.inv_t = 1.f / temperature, g.c = (float)(1.4426950408889634074 / (double)temperature);
    g.stats = stats, g.top_grad = top_grad, g.dloss = dloss, g.d = dlogits;
    return grad_any("mh_distill_topk_bwd", g, dtype, true, mh_stream(stream));
}

}  // extern "C"
