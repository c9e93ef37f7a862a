// Operators on rows of class scores x[0..k): log probabilities, entropy and the highest classes of a row, the
// divergence from a teacher's top classes, and their gradients.
//
// With c = log2(e) / T, m = max x and t_i = (x_i - m) c, everything follows from one pass over the row:
//     S = sum 2^t_i     U = sum 2^t_i t_i
//     ln p_i = ln2 (t_i - log2 S)        entropy = ln2 (log2 S - U / S)
// The pass keeps a running maximum per thread; when it rises by d (in units of t), S becomes S 2^-d and U becomes
// 2^-d (U - d S).  S, U and every statistic are held in 32 bits; the scores stay in the caller's type until they
// are in registers.
//
// Rows without a distribution: -inf scores have probability 0 and add nothing to U (0 log 0 = 0); a row of
// nothing but -inf has S = 0, log probability -inf everywhere, entropy 0 and gradient 0; a NaN or +inf among the
// scores makes S, and with it the row's results, NaN.
#include <algorithm>

#include "cd_internal.h"

namespace cd {

namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kInf = __builtin_inff();
// t is one fma, x c - fl(m c), while m c is small: what the rounding of m c leaves out is the same for every element of
// a row and cancels in p, but it has to stay far below 1.  From this magnitude on (and for a row masked with its type's
// lowest value throughout, where x c would overflow) the difference x - m is formed first.
constexpr float kPlainLimit = 0x1p20f;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 __attribute__((aligned(2))) u32x4_any;      // 16 bytes at any element's address

template <int TYPE> struct Elem;
template <> struct Elem<CD_T_F32> {
    static constexpr int kSize = 4, kVec = 4, kZeroBits = 0;        // (kZeroBits: low bits of a float that the type leaves 0)
    static constexpr uint32_t kNegInf = 0xff800000u;
    static __device__ __forceinline__ float load(const char* row, int64_t i) {
        return reinterpret_cast<const float*>(row)[i];
    }
    static __device__ __forceinline__ void store(char* row, int64_t i, float v) { reinterpret_cast<float*>(row)[i] = v; }
    static __device__ __forceinline__ void unpack(u32x4 w, float* x) {
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
    }
    static __device__ __forceinline__ u32x4 pack(const float* x) {
        u32x4 w;
        for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(x[i]);
        return w;
    }
};
template <> struct Elem<CD_T_BF16> {
    static constexpr int kSize = 2, kVec = 8, kZeroBits = 16;
    static constexpr uint32_t kNegInf = 0xff80ff80u;
    static __device__ __forceinline__ float load(const char* row, int64_t i) {
        return __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(row)[i] << 16);
    }
    static __device__ __forceinline__ void store(char* row, int64_t i, float v) {
        reinterpret_cast<__bf16*>(row)[i] = (__bf16)v;                    // round to nearest even
    }
    static __device__ __forceinline__ void unpack(u32x4 w, float* x) {
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float* x) {
        union { __bf16 h[8]; u32x4 w; } u;
        for (int i = 0; i < 8; ++i) u.h[i] = (__bf16)x[i];
        return u.w;
    }
};
template <> struct Elem<CD_T_F16> {
    static constexpr int kSize = 2, kVec = 8, kZeroBits = 13;
    static constexpr uint32_t kNegInf = 0xfc00fc00u;
    static __device__ __forceinline__ float load(const char* row, int64_t i) {
        return (float)reinterpret_cast<const _Float16*>(row)[i];
    }
    static __device__ __forceinline__ void store(char* row, int64_t i, float v) {
        reinterpret_cast<_Float16*>(row)[i] = (_Float16)v;                // round to nearest even
    }
    static __device__ __forceinline__ void unpack(u32x4 w, float* x) {
        union { u32x4 w; _Float16 h[8]; } u = {w};
        for (int i = 0; i < 8; ++i) x[i] = (float)u.h[i];
    }
    static __device__ __forceinline__ u32x4 pack(const float* x) {
        union { _Float16 h[8]; u32x4 w; } u;
        for (int i = 0; i < 8; ++i) u.h[i] = (_Float16)x[i];
        return u.w;
    }
};

// a score of a type known at run time: its bits, which the caller may leave in flight, and their value
__device__ __forceinline__ uint32_t load_bits(int type, const void* p, int64_t i) {
    return type == CD_T_F32 ? static_cast<const uint32_t*>(p)[i] : static_cast<const uint16_t*>(p)[i];
}
__device__ __forceinline__ float bits_value(int type, uint32_t b) {
    return type == CD_T_F32 ? __uint_as_float(b) : type == CD_T_BF16 ? __uint_as_float(b << 16)
         : (float)__builtin_bit_cast(_Float16, (uint16_t)b);
}
__device__ __forceinline__ float load_any(int type, const void* p, int64_t i) {
    return bits_value(type, load_bits(type, p, i));
}

// ---- wave reductions on the DPP network; the result is uniform ---------------------------------------------------
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp(float identity, float v) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(__float_as_uint(identity), __float_as_uint(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float lane_of(float v, int lane) {
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane));
}
__device__ __forceinline__ float wave_sum(float v) {      // a NaN in any lane makes the sum NaN
    v += dpp<0x111, 0xf>(0.f, v);                         // row_shr:1, 2, 4, 8: lane 15 of each row of 16 has its row
    v += dpp<0x112, 0xf>(0.f, v);
    v += dpp<0x114, 0xf>(0.f, v);
    v += dpp<0x118, 0xf>(0.f, v);
    v += dpp<0x142, 0xa>(0.f, v);                         // row_bcast:15 into rows 1 and 3
    v += dpp<0x143, 0xc>(0.f, v);                         // row_bcast:31 into rows 2 and 3
    return lane_of(v, 63);
}
__device__ __forceinline__ float wave_max(float v) {      // of numbers (a running maximum is never NaN)
    v = fmaxf(v, dpp<0x111, 0xf>(-kInf, v));
    v = fmaxf(v, dpp<0x112, 0xf>(-kInf, v));
    v = fmaxf(v, dpp<0x114, 0xf>(-kInf, v));
    v = fmaxf(v, dpp<0x118, 0xf>(-kInf, v));
    v = fmaxf(v, dpp<0x142, 0xa>(-kInf, v));
    v = fmaxf(v, dpp<0x143, 0xc>(-kInf, v));
    return lane_of(v, 63);
}

// ---- statistics of a row or a part of one ------------------------------------------------------------------------
struct Stat { float m, s, u; };     // maximum (-inf: nothing but -inf so far), S and U relative to it

__device__ __forceinline__ bool plain(float m, float c) { return fabsf(m * c) < kPlainLimit; }

// t of a score x against a maximum m; the same rounding everywhere, so that S and every p belong together
struct Ref {
    float c, mc, m;
    bool fast;
    __device__ __forceinline__ Ref(float m_, float c_) : c(c_) {
        fast = plain(m_, c_);
        m = m_ == -kInf ? 0.f : m_;
        mc = fast ? m_ * c_ : 0.f;
    }
    __device__ __forceinline__ float operator()(float x) const { return fast ? __builtin_fmaf(x, c, -mc) : (x - m) * c; }
};
// t of the maximum `from` against the maximum `to` >= from
__device__ __forceinline__ float shift(float from, float to, float c) {
    const bool f = plain(from, c), t = plain(to, c);      // (a plain maximum stands for fl(m c), another for m c itself)
    return f && t ? from * c - to * c
         : f ? __builtin_fmaf(-to, c, from * c) : t ? __builtin_fmaf(from, c, -(to * c)) : (from - to) * c;
}
__device__ __forceinline__ void rebase(Stat& a, float to, float c) {
    if (a.m != -kInf && a.m != to) {
        const float d = shift(a.m, to, c), f = __builtin_amdgcn_exp2f(d);
        a.u = f * __builtin_fmaf(fmaxf(d, -1e4f), a.s, a.u);
        a.s *= f;
    }
    a.m = to;
}

// (returns the largest of x, or NaN)  The terms of x are added among themselves before they join S and U: a long row of
// equal scores rounds every addition the same way, and a chain through all of them was off by 2e-4 in ln p at 16384 terms
// of a thread (65 x 2^24 bf16), where it is now one addition for N of them.  (Two chains per call would take two more
// registers, and with them a wave per SIMD of the 16-bit workgroup kernels: 4096 x 128000 bf16 201 us, with one 189.)
template <int N, bool ENT>
__device__ __forceinline__ float accumulate(const float* x, Stat& a, float c) {
    float cm = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) cm = __builtin_elementwise_maximum(cm, x[i]);
    if (cm > a.m) rebase(a, cm, c);                       // (not for a NaN: S becomes NaN below)
    const Ref t_of(a.m, c);
    float s = 0.f, u = 0.f;
    if (t_of.fast) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float t = __builtin_fmaf(x[i], c, -t_of.mc), e = __builtin_amdgcn_exp2f(t);
            s += e;
            if (ENT) u = __builtin_fmaf(e, fmaxf(t, -1e4f), u);     // the bound: 0 * -inf is 0 here
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float t = (x[i] - t_of.m) * c, e = __builtin_amdgcn_exp2f(t);
            s += e;
            if (ENT) u = __builtin_fmaf(e, fmaxf(t, -1e4f), u);
        }
    }
    a.s += s;
    if (ENT) a.u += u;
    return cm;
}

__device__ __forceinline__ Stat wave_merge(Stat a, float c) {
    const float m = wave_max(a.m);
    rebase(a, m, c);
    a.s = wave_sum(a.s);
    a.u = wave_sum(a.u);
    return a;
}

// ---- order of the classes of a row: 64-bit keys, larger = earlier (NaN, then by score, then by lower index) -----
__device__ __forceinline__ uint32_t score_key(float x) {
    if (x != x) return 0xfffffffeu;
    const uint32_t b = __float_as_uint(x + 0.f);          // -0 counts as +0
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_score(uint32_t k) {
    if (k == 0xfffffffeu) return __builtin_nanf("");
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ uint64_t full_key(float x, uint32_t index) {
    return (uint64_t)score_key(x) << 32 | (uint32_t)~index;
}
__device__ __forceinline__ uint64_t wave_max_key(uint64_t v) {
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t w = __shfl_xor((unsigned long long)v, o);
        v = w > v ? w : v;
    }
    return v;
}

// A row split between `parts` workgroups (grid y): part p has the scores [lo, hi), lo a multiple of 64.
struct Part { int lo, hi; };
__device__ __forceinline__ Part part_of(int k, int parts, int p) {
    const int64_t share = ((int64_t)(k + parts - 1) / parts + 63) / 64 * 64;
    return {(int)min((int64_t)k, share * p), (int)min((int64_t)k, share * (p + 1))};
}

// How a workgroup takes a row apart: `head` scores up to a 128-byte border (of the memory that counts most: the one
// written to, else the one read), vectors of 16 bytes, and the rest.  Thread j < extra has one score of head or rest.  Rows
// that begin anywhere cost 20 % more to read where the 16 bytes are not on a 4-byte border, and 15 to 20 % more to write
// where a wave's KB does not cover whole lines (2048 x 130001 bf16: 130 us against 107, gradient 293 against 242).
template <int TYPE> struct Grid {
    int head, nv, extra;
    __device__ __forceinline__ Grid(const char* border, int k) {
        head = min(k, (int)(-reinterpret_cast<uintptr_t>(border) & 127) / Elem<TYPE>::kSize);
        nv = (k - head) / Elem<TYPE>::kVec;
        extra = k - nv * Elem<TYPE>::kVec;
    }
    __device__ __forceinline__ int single(int j) const { return j < head ? j : j + nv * Elem<TYPE>::kVec; }
    __device__ __forceinline__ const u32x4_any* vectors(const char* x) const {
        return reinterpret_cast<const u32x4_any*>(x + head * Elem<TYPE>::kSize);
    }
    __device__ __forceinline__ u32x4_any* vectors(char* x) const {
        return reinterpret_cast<u32x4_any*>(x + head * Elem<TYPE>::kSize);
    }
};

struct LogProbsArgs {
    const char* x;
    int64_t n, row_bytes;
    int k, top;
    float c, t;
    const int64_t* ids;
    float *stats, *logp, *entropy, *top_logp;
    int64_t* top_ids;
    int parts;                      // of a row split between workgroups: what they find, [n][parts] and [n][parts][top]
    float4* part_stats;
    uint64_t* part_keys;
};

__device__ __forceinline__ float entropy_of(const Stat& a) {
    if (a.s == 0.f) return 0.f;
    const float h = kLn2 * (__builtin_amdgcn_logf(a.s) - a.u / a.s);
    return h < 0.f ? 0.f : h;
}
// ln p of a score; -inf in a row without a distribution
__device__ __forceinline__ float logp_of(float x, const Stat& a, float c, float temperature) {
    if (a.s == 0.f) return -kInf;
    const float t = Ref(a.m, c)(x);
    if (t < -1e30f && a.s == a.s) return (x - a.m) / temperature;       // in base 2 it could overflow; log S does not count
    const float lp = kLn2 * (t - __builtin_amdgcn_logf(a.s));
    return lp > 0.f ? 0.f : lp;
}

// the row's class id, -1 where it is skipped
__device__ __forceinline__ int id_of(const LogProbsArgs& A, int64_t row) {
    const int64_t id = A.ids ? A.ids[row] : -1;
    return id >= 0 && id < A.k ? (int)id : -1;
}
__device__ __forceinline__ void write_row(const LogProbsArgs& A, int64_t row, int id, float xid, const Stat& a) {
    A.stats[2 * row] = a.m;
    A.stats[2 * row + 1] = a.s;
    if (A.entropy) A.entropy[row] = entropy_of(a);
    if (A.logp) A.logp[row] = id >= 0 ? logp_of(xid, a, A.c, A.t) : 0.f;
}
__device__ __forceinline__ void write_top(const LogProbsArgs& A, int64_t row, int rank, uint64_t key, const Stat& a) {
    A.top_ids[row * A.top + rank] = (uint32_t)~(uint32_t)key;
    A.top_logp[row * A.top + rank] = logp_of(key_score((uint32_t)(key >> 32)), a, A.c, A.t);
}

// ================================================================================== one workgroup per row
// The highest classes of a row, from what the pass for the sums leaves behind.  The threads are 64 groups (256 for more
// than kFewTops alternatives), lane by lane over the waves, so that high scores side by side fall into different groups;
// the K-th largest of the groups' maxima, T, is at most the K-th largest score, since K groups have a score that high.
// Only threads whose own maximum reaches T can hold one of the K highest: about K (1 + K / 128), with 256 groups
// K (1 + K / 512), for scores in no particular order.  They read their scores again (from the caches; most of them only the
// piece that has their maximum), collect those that reach T in a list, and the list is ranked by counting.  Scores equal
// to T may be very many (a mask): where a wave finds more than kDense threads at T it leaves them, and the
// lowest-numbered classes at T are found by a scan in the order of the classes, which then ends early.  A list that
// overflows all the same, and NaN, take one scan per alternative, which is slow.  A list overflows where T is a mask's value
// and most threads of one wave have an allowed score besides their masked ones: that wave collects all of its masked scores.
// Then at least 40 groups have an allowed score, and fewer than there are alternatives: a short run of allowed classes and
// more than 40 alternatives (4096 x 128000 bf16, all but 400 consecutive classes at -inf: 189 us with 20 alternatives, 33 ms with 64).
constexpr int kDense = 24, kFewTops = 24;
template <int THREADS> struct BlockShared {
    static constexpr int kWaves = THREADS / 64, kList = 1024;
    float m[kWaves], s[kWaves], u[kWaves], total;
    uint32_t group[256];
    int count, above, dense, part[kWaves];
    uint8_t lane[kWaves][64];
    int piece[kWaves][64];
    uint64_t key[kWaves];
    uint64_t list[kList];
};

// the K-th largest of 64 lanes' keys, N to a lane
template <int ZERO_BITS, int N>
__device__ __forceinline__ uint32_t kth_key(const uint32_t (&key)[N], int K) {
    uint32_t t = 0, part[N];
#pragma unroll
    for (int i = 0; i < N; ++i) part[i] = key[i] >> ZERO_BITS;
    auto reach = [&](uint32_t v) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) c += __popcll(__ballot(part[i] >= v));
        return c >= K;
    };
    constexpr int kBits = 32 - ZERO_BITS;
    if (kBits & 1 && reach(1u << (kBits - 1))) t = 1u << (kBits - 1);
#pragma unroll
    for (int b = kBits / 2 * 2 - 2; b >= 0; b -= 2) {     // two bits a step: three counts that do not wait for one another
        const bool r1 = reach(t | 1u << b), r2 = reach(t | 2u << b), r3 = reach(t | 3u << b);
        t |= (r3 ? 3u : r2 ? 2u : r1 ? 1u : 0u) << b;
    }
    t <<= ZERO_BITS;
    return t & 0x80000000u ? t : t | ((1u << ZERO_BITS) - 1u);        // (keys of negative scores end in ones)
}

// The statistics of all threads' parts, the same bits in every thread; one barrier.  TOP: prepares block_top for that many
// alternatives (sh.group is 0 before).
template <bool TOP, int THREADS>
__device__ __forceinline__ Stat block_merge(Stat a, float c, BlockShared<THREADS>& sh, int top = 0) {
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    if (TOP) {
        atomicMax(&sh.group[top > kFewTops ? tid & 255 : lane], score_key(a.m));
        if (tid == 0) sh.count = sh.above = sh.dense = 0;
    }
    a = wave_merge(a, c);
    if (lane == 0) { sh.m[wave] = a.m; sh.s[wave] = a.s; sh.u[wave] = a.u; }
    __syncthreads();
    a.m = lane < THREADS / 64 ? sh.m[lane] : -kInf;
    a.s = lane < THREADS / 64 ? sh.s[lane] : 0.f;
    a.u = lane < THREADS / 64 ? sh.u[lane] : 0.f;
    return wave_merge(a, c);
}

// Where a thread's vectors have their largest score: in the piece of kPiece vectors of that number; `next` is the largest of
// its other pieces.
constexpr int kPiece = 4;
struct Peak { float m, next; int piece; };

// The calling thread's part of the pass over a row.
template <int TYPE, int THREADS, bool ENT>
__device__ __forceinline__ Stat block_pass(const char* x, int k, float c, Peak* peak) {
    using E = Elem<TYPE>;
    constexpr int VE = E::kVec, U = kPiece;
    const Grid<TYPE> g(x, k);
    const int tid = threadIdx.x;
    const u32x4_any* vec = g.vectors(x);
    Stat a = {-kInf, 0.f, 0.f};
    *peak = {-kInf, -kInf, 0};
    for (int v0 = 0; v0 < g.nv; v0 += U * THREADS) {
        float xs[U * VE];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            u32x4 w = {E::kNegInf, E::kNegInf, E::kNegInf, E::kNegInf};
            if (v0 + u * THREADS + tid < g.nv) w = vec[v0 + u * THREADS + tid];
            E::unpack(w, xs + u * VE);
        }
        const float cm = accumulate<U * VE, ENT>(xs, a, c);
        peak->next = fmaxf(peak->next, fminf(cm, peak->m));
        if (cm > peak->m) { peak->m = cm; peak->piece = v0; }
    }
    if (tid < g.extra) {
        const float xt = E::load(x, g.single(tid));
        accumulate<1, ENT>(&xt, a, c);
    }
    return a;
}

// Calls emit(rank, key) for the K highest of the k scores, every rank once, by any thread.
template <int TYPE, int THREADS, class Emit>
__device__ __forceinline__ void block_top(const char* x, int k, int K, const Peak& peak, bool nan, BlockShared<THREADS>& sh,
                                          Emit emit) {
    using E = Elem<TYPE>;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const Grid<TYPE> g(x, k);
    uint32_t T;
    if (K > kFewTops) {
        const uint32_t key[4] = {sh.group[lane], sh.group[lane + 64], sh.group[lane + 128], sh.group[lane + 192]};
        T = kth_key<E::kZeroBits, 4>(key, K);
    } else {
        const uint32_t key[1] = {sh.group[lane]};
        T = kth_key<E::kZeroBits, 1>(key, K);
    }
    if (!nan) {
        const float xt = key_score(T);
        auto collect = [&](float v, uint32_t i, bool ties) {
            if (ties ? v >= xt : v > xt) {
                const int at = atomicAdd(&sh.count, 1);
                if (at < sh.kList) sh.list[at] = full_key(v, i);
                if (v > xt) atomicAdd(&sh.above, 1);
            }
        };
        const bool dense = __popcll(__ballot(peak.m == xt)) > kDense;
        if (dense && lane == 0) sh.dense = 1;
        // threads that look into one piece, then threads that look into all of theirs; a lane per vector
        const bool take = dense ? peak.m > xt : peak.m >= xt, more = dense ? peak.next > xt : peak.next >= xt;
        auto look = [&](bool mine, int pieces) {
            const uint64_t who = __ballot(mine);
            if (mine) {
                const int at = __popcll(who & ((1ull << lane) - 1));
                sh.lane[wave][at] = lane;
                sh.piece[wave][at] = pieces == 1 ? peak.piece : 0;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            const int share = pieces * kPiece, items = __popcll(who) * share;
            for (int it = lane; it < items; it += 64) {
                const int q = it / share, v = sh.piece[wave][q] + (it - q * share) * THREADS + wave * 64 + sh.lane[wave][q];
                if (v < g.nv) {
                    float xs[E::kVec];
                    E::unpack(g.vectors(x)[v], xs);
#pragma unroll
                    for (int i = 0; i < E::kVec; ++i) collect(xs[i], g.head + v * E::kVec + i, !dense);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        };
        look(take && !more, 1);
        if (__any(take && more)) look(take && more, (g.nv + kPiece * THREADS - 1) / (kPiece * THREADS));
        if (tid < g.extra) collect(E::load(x, g.single(tid)), g.single(tid), !dense);
    }
    __syncthreads();
    for (int i = tid; i < 256; i += THREADS) sh.group[i] = 0;     // for the next row, which begins behind a barrier
    const int count = sh.count, above = sh.above, dense = sh.dense;
    if (!nan && count <= sh.kList) {
        for (int e = tid; e < count; e += THREADS) {
            const uint64_t key = sh.list[e];
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < count; ++j) rank += sh.list[j] > key;
            if (rank < K && (!dense || (uint32_t)(key >> 32) > T)) emit(rank, key);
        }
        for (int base = 0, rank = above; dense && rank < K && base < k; base += THREADS) {
            const int i = base + tid;
            const bool hit = i < k && score_key(E::load(x, i)) == T;
            const uint64_t hits = __ballot(hit);
            if (lane == 0) sh.part[wave] = __popcll(hits);
            __syncthreads();
            int before = 0, all = 0;
            for (int w = 0; w < THREADS / 64; ++w) {
                before += w < wave ? sh.part[w] : 0;
                all += sh.part[w];
            }
            const int at = rank + before + __popcll(hits & ((1ull << lane) - 1));
            if (hit && at < K) emit(at, (uint64_t)T << 32 | (uint32_t)~i);
            rank += all;
            __syncthreads();
        }
        return;
    }
    uint64_t last = ~0ull;
    for (int r = 0; r < K; ++r) {                         // the largest key below the last one found
        uint64_t best = 0;
        for (int i = tid; i < k; i += THREADS) {
            const uint64_t key = full_key(E::load(x, i), i);
            if (key < last && key > best) best = key;
        }
        best = wave_max_key(best);
        if (lane == 0) sh.key[wave] = best;
        __syncthreads();
        for (int w = 0; w < THREADS / 64; ++w) best = sh.key[w] > best ? sh.key[w] : best;
        if (tid == 0) emit(r, best);
        last = best;
        __syncthreads();
    }
}

template <int TYPE, int THREADS, bool ENT>
__global__ __launch_bounds__(THREADS) void log_probs_block_kernel(LogProbsArgs A) {
    __shared__ BlockShared<THREADS> sh;
    for (int i = threadIdx.x; i < 256; i += THREADS) sh.group[i] = 0;
    __syncthreads();
    for (int64_t row = blockIdx.x; row < A.n; row += gridDim.x) {
        const char* x = A.x + row * A.row_bytes;
        const int id = id_of(A, row);
        Peak peak;
        const Stat own = block_pass<TYPE, THREADS, ENT>(x, A.k, A.c, &peak);
        const float xid = id >= 0 && threadIdx.x == 0 ? Elem<TYPE>::load(x, id) : 0.f;
        const Stat a = block_merge<true>(own, A.c, sh, A.top);
        if (threadIdx.x == 0) write_row(A, row, id, xid, a);
        if (A.top)
            block_top<TYPE>(x, A.k, A.top, peak, a.s != a.s, sh,
                            [&](int rank, uint64_t key) { write_top(A, row, rank, key, a); });
        __syncthreads();
    }
}

// Few, long rows: several workgroups per row leave their statistics and highest classes in the workspace, and one
// workgroup per row joins them.
template <int TYPE, int THREADS, bool ENT>
__global__ __launch_bounds__(THREADS) void log_probs_part_kernel(LogProbsArgs A) {
    __shared__ BlockShared<THREADS> sh;
    const int64_t row = blockIdx.x, slot = row * A.parts + blockIdx.y;
    const Part p = part_of(A.k, A.parts, blockIdx.y);
    const int have = min(A.top, p.hi - p.lo);
    const char* x = A.x + row * A.row_bytes + (int64_t)p.lo * Elem<TYPE>::kSize;
    for (int i = threadIdx.x; i < 256; i += THREADS) sh.group[i] = 0;
    __syncthreads();
    Peak peak;
    const Stat a = block_merge<true>(block_pass<TYPE, THREADS, ENT>(x, p.hi - p.lo, A.c, &peak), A.c, sh, have);
    if (threadIdx.x == 0) A.part_stats[slot] = {a.m, a.s, a.u, 0.f};
    if (A.top) {
        uint64_t* keys = A.part_keys + slot * A.top;
        for (int r = have + threadIdx.x; r < A.top; r += THREADS) keys[r] = 0;
        if (have) block_top<TYPE>(x, p.hi - p.lo, have, peak, a.s != a.s, sh,
                                  [&](int rank, uint64_t key) { keys[rank] = key - p.lo; });
    }
}
__device__ __forceinline__ Stat join_stats(const float4* part, int parts, float c) {
    const int lane = threadIdx.x & 63;
    Stat a = {-kInf, 0.f, 0.f};
    if (lane < parts) { const float4 v = part[lane]; a = {v.x, v.y, v.z}; }
    return wave_merge(a, c);
}
// A bound as in block_top, from the first keys of every part, 64 N in all.
template <int N>
__device__ __forceinline__ uint64_t join_bound(const uint64_t* keys, int parts, int top) {
    const int lane = threadIdx.x & 63, heads = 64 * N / parts;
    uint64_t mine[N];
    uint32_t high[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int q = (lane + 64 * j) / heads, r = lane + 64 * j - q * heads;
        mine[j] = q < parts && r < top ? keys[q * top + r] : 0;
        high[j] = (uint32_t)(mine[j] >> 32);
    }
    auto reach = [&](uint64_t v) {
        int c = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) c += __popcll(__ballot(mine[j] >= v));
        return c;
    };
    uint64_t t = (uint64_t)kth_key<0, N>(high, top) << 32;
    if (reach(t) >= top + 16)                             // many equal scores: the classes count as well
        for (int b = 31; b >= 0; --b)
            if (reach(t | 1ull << b) >= top) t |= 1ull << b;
    return t;
}
template <int TYPE>
__global__ __launch_bounds__(256) void log_probs_join_kernel(LogProbsArgs A) {
    __shared__ uint64_t list[64 * kMaxTop];
    __shared__ int count;
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const int id = id_of(A, row);
    const float xid = id >= 0 ? Elem<TYPE>::load(A.x + row * A.row_bytes, id) : 0.f;
    const Stat a = join_stats(A.part_stats + row * A.parts, A.parts, A.c);
    if (tid == 0) write_row(A, row, id, xid, a);
    if (!A.top) return;
    if (tid == 0) count = 0;
    __syncthreads();
    const uint64_t* keys = A.part_keys + row * A.parts * A.top;
    const uint64_t t = A.top > kFewTops ? join_bound<4>(keys, A.parts, A.top) : join_bound<1>(keys, A.parts, A.top);
#pragma unroll 4
    for (int e = tid; e < A.parts * A.top; e += 256) {
        const uint64_t key = keys[e];
        if (key != 0 && key >= t) list[atomicAdd(&count, 1)] = key;       // (in any order: they are ranked)
    }
    __syncthreads();
    for (int e = tid; e < count; e += 256) {
        const uint64_t key = list[e];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < count; ++j) rank += list[j] > key;
        if (rank < A.top) write_top(A, row, rank, key, a);
    }
}

// Writes f(score) for every score of a row, backwards: what the pass before has read last is in the caches, and the
// writes go past them (4096 x 131072 bf16 as the second half of distill: 570 us with ordinary stores, 525 so; forwards
// 587 and 569).  dx may be x itself.
template <int TYPE, int THREADS, class F>
__device__ __forceinline__ void sweep(const char* x, char* dx, int k, F f) {
    using E = Elem<TYPE>;
    constexpr int U = 4, VE = E::kVec;
    const Grid<TYPE> g(dx, k);
    const int tid = threadIdx.x;
    const u32x4_any* from = g.vectors(x);
    u32x4_any* to = g.vectors(dx);
    if (tid < g.extra) E::store(dx, g.single(tid), f(E::load(x, g.single(tid))));
    for (int v0 = (g.nv - 1) / (U * THREADS) * (U * THREADS); v0 >= 0; v0 -= U * THREADS) {
        u32x4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (v0 + u * THREADS + tid < g.nv) w[u] = from[v0 + u * THREADS + tid];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float d[VE];
            E::unpack(w[u], d);
#pragma unroll
            for (int i = 0; i < VE; ++i) d[i] = f(d[i]);
            if (v0 + u * THREADS + tid < g.nv) __builtin_nontemporal_store(E::pack(d), to + v0 + u * THREADS + tid);
        }
    }
}
// Zeroes a row.
template <int TYPE, int THREADS>
__device__ __forceinline__ void clear(char* dx, int k) {
    const Grid<TYPE> g(dx, k);
    const int tid = threadIdx.x;
    for (int v = tid; v < g.nv; v += THREADS) __builtin_nontemporal_store(u32x4{0, 0, 0, 0}, g.vectors(dx) + v);
    if (tid < g.extra) Elem<TYPE>::store(dx, g.single(tid), 0.f);
}

// ---- gradients ---------------------------------------------------------------------------------------------------
// d(g_l ln p_id + g_h entropy) / dx_i = [g_l (i == id) - p_i (g_l + g_h (ln p_i + entropy))] / T
struct LogProbsGradArgs {
    const char* x;
    char* dx;
    int64_t n, row_bytes, dx_row_bytes;
    int k;
    float c, inv_t;
    const int64_t* ids;
    const float *stats, *entropy, *g_logp, *g_entropy;
};
// dx_i = 2^t_i (a + b t_i), plus hit at class id; `on` is false where no gradient arrives (the end of a padded batch), or the
// row has no distribution: 0 then, whatever the scores
struct GradRow { float a, b, hit; int id; bool on; };
__device__ __forceinline__ GradRow grad_row(const LogProbsGradArgs& A, int64_t row, float s) {
    const int64_t id = A.ids ? A.ids[row] : -1;
    const bool labelled = id >= 0 && id < A.k;
    const float gl = labelled && A.g_logp ? A.g_logp[row] : 0.f, gh = A.g_entropy ? A.g_entropy[row] : 0.f;
    GradRow g = {0.f, 0.f, 0.f, -1, s != 0.f && (gl != 0.f || gh != 0.f)};
    if (!g.on) return g;
    const float inv = A.inv_t / s;
    g.b = -gh * kLn2 * inv;
    g.a = -(gl + gh * ((A.g_entropy ? A.entropy[row] : 0.f) - kLn2 * __builtin_amdgcn_logf(s))) * inv;
    g.hit = gl * A.inv_t;
    g.id = labelled ? (int)id : -1;
    return g;
}
// (of a row that is on)
__device__ __forceinline__ float grad_of(float t, const GradRow& g) {
    return __builtin_amdgcn_exp2f(t) * __builtin_fmaf(g.b, fmaxf(t, -1e4f), g.a);
}

template <int TYPE, int THREADS>
__global__ __launch_bounds__(THREADS) void log_probs_grad_kernel(LogProbsGradArgs A) {
    const Part p = part_of(A.k, gridDim.y, blockIdx.y);
    for (int64_t back = blockIdx.x; back < A.n; back += gridDim.x) {
        const int64_t row = A.n - 1 - back;               // the rows that the forward call has read last come first
        const float m = A.stats[2 * row], s = A.stats[2 * row + 1];
        const GradRow g = grad_row(A, row, s);
        const Ref t_of(m, A.c);
        const char* x = A.x + row * A.row_bytes + (int64_t)p.lo * Elem<TYPE>::kSize;
        char* dx = A.dx + row * A.dx_row_bytes + (int64_t)p.lo * Elem<TYPE>::kSize;
        const bool here = g.id >= p.lo && g.id < p.hi;
        const float hit = here ? grad_of(t_of(Elem<TYPE>::load(x, g.id - p.lo)), g) + g.hit : 0.f;
        __syncthreads();                                  // (dx may be x)
        if (!g.on) clear<TYPE, THREADS>(dx, p.hi - p.lo);
        else if (t_of.fast) sweep<TYPE, THREADS>(x, dx, p.hi - p.lo, [&](float v) { return grad_of(__builtin_fmaf(v, A.c, -t_of.mc), g); });
        else sweep<TYPE, THREADS>(x, dx, p.hi - p.lo, [&](float v) { return grad_of(t_of(v), g); });
        __syncthreads();                                  // the row first, then its class
        if (threadIdx.x == 0 && here) Elem<TYPE>::store(dx, g.id - p.lo, hit);
    }
}

// ================================================================================== distillation
// q = softmax(teacher / T) over the used entries;  loss = w T^2 sum_j q_j (ln q_j - ln p_id_j)
// dx_i = w T (p_i - sum of q_j with id_j = i)
struct DistillArgs {
    const char* x;
    char* dx;                       // NULL: the loss alone
    int64_t n, row_bytes, dx_row_bytes;
    int k, entries, teacher_type;
    float c, t;
    const int64_t* ids;
    const void* teacher;
    const float *weights, *g_loss;  // g_loss: only the gradient, each row's times g_loss
    float *stats, *loss;
    int parts;                      // of a row split between workgroups: what they find, [n][parts], and the student's
    float4* part_stats;             // scores of the entries [n][entries]
    float* part_x;
};
template <int PER> struct Teacher { // the entries of one row, spread over a wave: entry lane + 64 e, e < PER
    int64_t raw_id[PER];            // as loaded
    uint32_t raw_score[PER];
    int id[PER];                    // -1: unused
    float lq[PER];                  // log2 q
    float q[PER];
    float sum[PER];                 // of a class named more than once: its q's together at its first entry, else -1
    float x[PER];                   // the student's score
    float total;                    // sum of 2^(..) before normalising: 0 where no entry counts
};
template <int PER>
__device__ __forceinline__ void load_entries(Teacher<PER>& r, const DistillArgs& A, int64_t row) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int j = lane + 64 * e;
        r.raw_id[e] = -1;
        r.raw_score[e] = 0;
        if (j < A.entries) {
            r.raw_id[e] = A.ids[row * A.entries + j];
            r.raw_score[e] = load_bits(A.teacher_type, A.teacher, row * A.entries + j);
        }
    }
}
template <int PER>
__device__ __forceinline__ void share_out(Teacher<PER>& r, const DistillArgs& A) {
    const int lane = threadIdx.x & 63;
    float m = -kInf, total = 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const bool used = r.raw_id[e] >= 0 && r.raw_id[e] < A.k;
        r.id[e] = used ? (int)r.raw_id[e] : -1;
        r.lq[e] = used ? bits_value(A.teacher_type, r.raw_score[e]) : -kInf;
        m = fmaxf(m, r.lq[e]);
    }
    m = wave_max(m);
    const Ref t_of(m, A.c);
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        r.lq[e] = t_of(r.lq[e]);
        r.q[e] = r.id[e] >= 0 ? __builtin_amdgcn_exp2f(r.lq[e]) : 0.f;
        total += r.q[e];
    }
    r.total = wave_sum(total);
    const float l = __builtin_amdgcn_logf(r.total), inv = 1.f / r.total;
#pragma unroll
    for (int e = 0; e < PER; ++e) { r.lq[e] -= l; r.q[e] *= inv; r.sum[e] = r.id[e] >= 0 ? r.q[e] : -1.f; }
    if (!A.dx) return;
    // entries of the same class: same[e][f] are the lanes whose entry f names the class of this lane's entry e, found bit
    // by bit of the class
    uint64_t same[PER][PER];
#pragma unroll
    for (int e = 0; e < PER; ++e)
#pragma unroll
        for (int f = 0; f < PER; ++f) same[e][f] = __ballot(r.id[f] >= 0);
    for (int b = 0; (A.k - 1) >> b; ++b)
#pragma unroll
        for (int f = 0; f < PER; ++f) {
            const uint64_t ones = __ballot(r.id[f] >> b & 1);
#pragma unroll
            for (int e = 0; e < PER; ++e) same[e][f] &= r.id[e] >> b & 1 ? ones : ~ones;
        }
    bool again = false;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        int count = 0;
#pragma unroll
        for (int f = 0; f < PER; ++f) count += __popcll(same[e][f]);
        again |= r.id[e] >= 0 && count > 1;
    }
    if (!__any(again)) return;                            // no class twice
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        float sum = 0.f;
        bool first = r.id[e] >= 0;
#pragma unroll
        for (int f = 0; f < PER; ++f) {
            if (first && (f < e ? same[e][f] != 0 : f == e && (same[e][e] & ((1ull << lane) - 1)))) first = false;
            for (uint64_t left = r.id[e] >= 0 ? same[e][f] : 0; __any(left != 0); left &= left - 1) {
                const float q = __shfl(r.q[f], left ? __ffsll((unsigned long long)left) - 1 : lane);
                if (left) sum += q;
            }
        }
        r.sum[e] = first ? sum : -1.f;
    }
}
template <int TYPE, int PER>
__device__ __forceinline__ void load_student(Teacher<PER>& r, const char* x, Part p) {
#pragma unroll
    for (int e = 0; e < PER; ++e) r.x[e] = r.id[e] >= p.lo && r.id[e] < p.hi ? Elem<TYPE>::load(x, r.id[e]) : 0.f;
}
// one entry's part of a loss of weight and temperature 1
__device__ __forceinline__ float loss_term(float q, float lq, float x, const Stat& a, float c, float temperature) {
    return q != 0.f ? q * (kLn2 * lq - logp_of(x, a, c, temperature)) : 0.f;
}
// the row's loss, uniform over the wave
template <int PER>
__device__ __forceinline__ float teacher_loss(const Teacher<PER>& r, const Stat& a, const DistillArgs& A, float w) {
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e)
        if (r.id[e] >= 0) sum += loss_term(r.q[e], r.lq[e], r.x[e], a, A.c, A.t);
    return w * (A.t * A.t) * wave_sum(sum);
}
// the gradient at the teacher's classes, over what the sweep has written there
template <int TYPE, int PER>
__device__ __forceinline__ void fix_gradient(const Teacher<PER>& r, const Stat& a, const DistillArgs& A, float w, char* dx,
                                             Part p) {
    const Ref t_of(a.m, A.c);
    const float inv = 1.f / a.s;
#pragma unroll
    for (int e = 0; e < PER; ++e)
        if (!(r.sum[e] < 0.f) && r.id[e] >= p.lo && r.id[e] < p.hi)
            Elem<TYPE>::store(dx, r.id[e], w * A.t * (__builtin_amdgcn_exp2f(t_of(r.x[e])) * inv - r.sum[e]));
}

// w T p of every class of a part
template <int TYPE, int THREADS>
__device__ __forceinline__ void distill_sweep(const DistillArgs& A, int64_t row, Part p, const Stat& a, float w) {
    const char* x = A.x + row * A.row_bytes + (int64_t)p.lo * Elem<TYPE>::kSize;
    char* dx = A.dx + row * A.dx_row_bytes + (int64_t)p.lo * Elem<TYPE>::kSize;
    const Ref t_of(a.m, A.c);
    const float f = w * A.t / a.s;
    if (t_of.fast)
        sweep<TYPE, THREADS>(x, dx, p.hi - p.lo, [&](float v) { return f * __builtin_amdgcn_exp2f(__builtin_fmaf(v, A.c, -t_of.mc)); });
    else
        sweep<TYPE, THREADS>(x, dx, p.hi - p.lo, [&](float v) { return f * __builtin_amdgcn_exp2f(t_of(v)); });
}

// What the kernels below share: the row's weight, its teacher (wave 0; every thread learns whether an entry counts), its
// statistics from `pass`, the loss (part 0), and the gradient of part p from `grad(w, a)`, which writes w T p of every
// class.  `load` may start loads that `pass` uses; `student` loads the student's scores of the teacher's classes.
template <int TYPE, int THREADS, int PER, class Load, class Student, class Pass, class Grad>
__device__ __forceinline__ void distill_row(const DistillArgs& A, int64_t row, Part p, BlockShared<THREADS>& sh,
                                            Load load, Student student, Pass pass, Grad grad) {
    char* dx = A.dx + row * A.dx_row_bytes;
    const int tid = threadIdx.x;
    float w = A.weights ? A.weights[row] : 1.f;
    if (A.g_loss && w != 0.f) w *= A.g_loss[row];
    Stat a = {-kInf, 0.f, 0.f};
    Teacher<PER> te;
    bool on = false;
    if (w != 0.f) {
        if (tid < 64) load_entries<PER>(te, A, row);      // (in flight before the row's own loads, if `load` makes them)
        load();
        if (tid < 64) {
            share_out<PER>(te, A);
            student(te);
            if (tid == 0) sh.total = te.total;
        }
        a = pass();                                       // (has a barrier: all of x has been read that is read here)
        on = sh.total != 0.f;
    }
    if (A.loss && p.lo == 0 && tid < 64) {
        const float loss = on ? teacher_loss<PER>(te, a, A, w) : 0.f;
        if (tid == 0) {
            A.loss[row] = loss;
            A.stats[2 * row] = a.m;
            A.stats[2 * row + 1] = a.s;
        }
    }
    if (A.dx) {
        const bool live = on && a.s != 0.f;
        if (live) grad(w, a);
        else clear<TYPE, THREADS>(dx + (int64_t)p.lo * Elem<TYPE>::kSize, p.hi - p.lo);
        __syncthreads();                                  // the row first, then the teacher's classes
        if (live && tid < 64) fix_gradient<TYPE, PER>(te, a, A, w, dx, p);
    }
    __syncthreads();
}

template <int TYPE, int THREADS, int PER>
__global__ __launch_bounds__(THREADS) void distill_block_kernel(DistillArgs A) {
    __shared__ BlockShared<THREADS> sh;
    const Part all = {0, A.k};
    for (int64_t row = blockIdx.x; row < A.n; row += gridDim.x) {
        const char* x = A.x + row * A.row_bytes;
        distill_row<TYPE, THREADS, PER>(A, row, all, sh, [] {},
            [&](Teacher<PER>& te) { load_student<TYPE, PER>(te, x, all); },
            [&] {
                Peak peak;
                return block_merge<false>(block_pass<TYPE, THREADS, false>(x, A.k, A.c, &peak), A.c, sh);
            },
            [&](float w, const Stat& a) { distill_sweep<TYPE, THREADS>(A, row, all, a, w); });
    }
}

// Few, long rows, as in log_probs: the parts' statistics first, then loss and gradient, part by part again.
template <int TYPE, int THREADS>
__global__ __launch_bounds__(THREADS) void distill_part_kernel(DistillArgs A) {
    __shared__ BlockShared<THREADS> sh;
    const int64_t row = blockIdx.x;
    if (A.weights && A.weights[row] == 0.f) return;
    const Part p = part_of(A.k, A.parts, blockIdx.y);
    const char* x = A.x + row * A.row_bytes;
    const int j = threadIdx.x;
    if (blockIdx.y == 0 && j < A.entries) {               // before the gradient, which may take the scores' place
        const int64_t id = A.ids[row * A.entries + j];
        A.part_x[row * A.entries + j] = id >= 0 && id < A.k ? Elem<TYPE>::load(x, id) : 0.f;
    }
    Peak peak;
    const Stat a = block_merge<false>(
        block_pass<TYPE, THREADS, false>(x + (int64_t)p.lo * Elem<TYPE>::kSize, p.hi - p.lo, A.c, &peak), A.c, sh);
    if (threadIdx.x == 0) A.part_stats[row * A.parts + blockIdx.y] = {a.m, a.s, 0.f, 0.f};
}
template <int TYPE, int THREADS, int PER>
__global__ __launch_bounds__(THREADS) void distill_join_kernel(DistillArgs A) {
    __shared__ BlockShared<THREADS> sh;
    const int64_t row = blockIdx.x;
    const Part p = part_of(A.k, gridDim.y, blockIdx.y);   // (grid y is 1 where there is no gradient)
    distill_row<TYPE, THREADS, PER>(A, row, p, sh, [] {},
        [&](Teacher<PER>& te) {
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const int j = (threadIdx.x & 63) + 64 * e;
                te.x[e] = j < A.entries ? A.part_x[row * A.entries + j] : 0.f;
            }
        },
        [&] {
            __syncthreads();
            return join_stats(A.part_stats + row * A.parts, A.parts, A.c);
        },
        [&](float w, const Stat& a) { distill_sweep<TYPE, THREADS>(A, row, p, a, w); });
}

// Loss and gradient of rows that fit the threads' registers, V vectors each: they are read once, all loads at once, and
// the second half of the work starts from the registers.
template <int TYPE, int THREADS, int V, int PER>
__global__ __launch_bounds__(THREADS) void distill_held_kernel(DistillArgs A) {
    using E = Elem<TYPE>;
    constexpr int VE = E::kVec, U = 2;
    __shared__ BlockShared<THREADS> sh;
    const int tid = threadIdx.x;
    const Part all = {0, A.k};
    for (int64_t row = blockIdx.x; row < A.n; row += gridDim.x) {
        const char* x = A.x + row * A.row_bytes;
        char* dx = A.dx + row * A.dx_row_bytes;
        const Grid<TYPE> g(dx, A.k);
        const char* from = x + g.head * E::kSize;
        char* to = dx + g.head * E::kSize;
        u32x4 w[V];
        float single = -kInf;
        distill_row<TYPE, THREADS, PER>(A, row, all, sh,
            [&] {
#pragma unroll
                for (int u = 0; u < V; ++u) {
                    w[u] = u32x4{E::kNegInf, E::kNegInf, E::kNegInf, E::kNegInf};
                    if (u * THREADS + tid < g.nv) w[u] = reinterpret_cast<const u32x4_any*>(from + 16 * u * THREADS)[tid];
                }
                if (tid < g.extra) single = E::load(x, g.single(tid));
            },
            [&](Teacher<PER>& te) { load_student<TYPE, PER>(te, x, all); },
            [&] {
                Stat a = {-kInf, 0.f, 0.f};
#pragma unroll
                for (int u = 0; u < V; u += U) {
                    float xs[U * VE];
#pragma unroll
                    for (int i = 0; i < U; ++i) E::unpack(w[u + i], xs + i * VE);
                    accumulate<U * VE, false>(xs, a, A.c);
                }
                accumulate<1, false>(&single, a, A.c);
                return block_merge<false>(a, A.c, sh);
            },
            [&](float weight, const Stat& a) {
                const Ref t_of(a.m, A.c);
                const float f = weight * A.t / a.s;
#pragma unroll
                for (int u = 0; u < V; ++u) {
                    float d[VE];
                    E::unpack(w[u], d);
                    if (t_of.fast) {
#pragma unroll
                        for (int i = 0; i < VE; ++i) d[i] = f * __builtin_amdgcn_exp2f(__builtin_fmaf(d[i], A.c, -t_of.mc));
                    } else {
                        for (int i = 0; i < VE; ++i) d[i] = f * __builtin_amdgcn_exp2f(t_of(d[i]));
                    }
                    if (u * THREADS + tid < g.nv)
                        __builtin_nontemporal_store(E::pack(d), reinterpret_cast<u32x4_any*>(to + 16 * u * THREADS) + tid);
                }
                if (tid < g.extra) E::store(dx, g.single(tid), f * __builtin_amdgcn_exp2f(t_of(single)));
            });
    }
}

// the gradient alone, from the statistics of the forward call
template <int TYPE, int THREADS, int PER>
__global__ __launch_bounds__(THREADS) void distill_grad_kernel(DistillArgs A) {
    __shared__ BlockShared<THREADS> sh;
    const Part p = part_of(A.k, gridDim.y, blockIdx.y);
    for (int64_t back = blockIdx.x; back < A.n; back += gridDim.x) {
        const int64_t row = A.n - 1 - back;
        distill_row<TYPE, THREADS, PER>(A, row, p, sh, [] {},
            [&](Teacher<PER>& te) { load_student<TYPE, PER>(te, A.x + row * A.row_bytes, p); },
            [&] {
                __syncthreads();
                return Stat{A.stats[2 * row], A.stats[2 * row + 1], 0.f};
            },
            [&](float w, const Stat& a) { distill_sweep<TYPE, THREADS>(A, row, p, a, w); });
    }
}

// ================================================================================== one thread per row, up to 16 scores
constexpr int kThreadClasses = 16;

template <int TYPE, int K>
__device__ __forceinline__ void load_short(const char* x, int k, float* v) {
#pragma unroll
    for (int i = 0; i < K; ++i) v[i] = i < k ? Elem<TYPE>::load(x, i) : -kInf;
}

template <int TYPE, int K>
__global__ __launch_bounds__(64) void log_probs_thread_kernel(LogProbsArgs A) {
    for (int64_t row = (int64_t)blockIdx.x * 64 + threadIdx.x; row < A.n; row += (int64_t)gridDim.x * 64) {
        const char* x = A.x + row * A.row_bytes;
        float v[K];
        load_short<TYPE, K>(x, A.k, v);
        Stat a = {-kInf, 0.f, 0.f};
        accumulate<K, true>(v, a, A.c);
        const int id = id_of(A, row);
        float xid = 0.f;
#pragma unroll
        for (int i = 0; i < K; ++i) if (i == id) xid = v[i];
        write_row(A, row, id, xid, a);
        uint32_t key[K], used = 0;
#pragma unroll
        for (int i = 0; i < K; ++i) key[i] = score_key(v[i]);
        for (int r = 0; r < A.top; ++r) {
            uint32_t best = 0;
            int at = 0;
#pragma unroll
            for (int i = 0; i < K; ++i)
                if (i < A.k && !(used >> i & 1) && key[i] > best) { best = key[i]; at = i; }
            used |= 1u << at;
            write_top(A, row, r, (uint64_t)best << 32 | (uint32_t)~at, a);
        }
    }
}

template <int TYPE, int K>
__global__ __launch_bounds__(64) void log_probs_grad_thread_kernel(LogProbsGradArgs A) {
    for (int64_t row = (int64_t)blockIdx.x * 64 + threadIdx.x; row < A.n; row += (int64_t)gridDim.x * 64) {
        const float m = A.stats[2 * row], s = A.stats[2 * row + 1];
        float v[K];
        load_short<TYPE, K>(A.x + row * A.row_bytes, A.k, v);
        const GradRow g = grad_row(A, row, s);
        const Ref t_of(m, A.c);
#pragma unroll
        for (int i = 0; i < K; ++i)
            if (i < A.k)
                Elem<TYPE>::store(A.dx + row * A.dx_row_bytes, i,
                                  g.on ? grad_of(t_of(v[i]), g) + (i == g.id ? g.hit : 0.f) : 0.f);
    }
}

template <int TYPE, int K>
__global__ __launch_bounds__(64) void distill_thread_kernel(DistillArgs A) {
    for (int64_t row = (int64_t)blockIdx.x * 64 + threadIdx.x; row < A.n; row += (int64_t)gridDim.x * 64) {
        const char* x = A.x + row * A.row_bytes;
        float w = A.weights ? A.weights[row] : 1.f;
        if (A.g_loss && w != 0.f) w *= A.g_loss[row];
        float v[K], qk[K], loss = 0.f, total = 0.f;
        Stat a = {-kInf, 0.f, 0.f};
        if (w != 0.f) {
            load_short<TYPE, K>(x, A.k, v);
            accumulate<K, false>(v, a, A.c);
            const int64_t* ids = A.ids + row * A.entries;
            auto used = [&](int64_t id) { return id >= 0 && id < A.k; };
            auto score = [&](int j) { return load_any(A.teacher_type, A.teacher, row * A.entries + j); };
            float m = -kInf;
            for (int j = 0; j < A.entries; ++j) if (used(ids[j])) m = fmaxf(m, score(j));
            const Ref t_of(m, A.c);
            for (int j = 0; j < A.entries; ++j) if (used(ids[j])) total += __builtin_amdgcn_exp2f(t_of(score(j)));
            const float l = __builtin_amdgcn_logf(total), inv = 1.f / total;
#pragma unroll
            for (int i = 0; i < K; ++i) qk[i] = 0.f;
            if (total != 0.f)
                for (int j = 0; j < A.entries; ++j) {
                    const int64_t id = ids[j];
                    if (!used(id)) continue;
                    const float t = t_of(score(j)), q = __builtin_amdgcn_exp2f(t) * inv;
                    float xj = 0.f;
#pragma unroll
                    for (int i = 0; i < K; ++i) if (i == id) { xj = v[i]; qk[i] += q; }
                    loss += loss_term(q, t - l, xj, a, A.c, A.t);
                }
        }
        const bool on = w != 0.f && total != 0.f, live = on && a.s != 0.f;
        if (A.loss) {
            A.loss[row] = on ? w * (A.t * A.t) * loss : 0.f;
            A.stats[2 * row] = a.m;
            A.stats[2 * row + 1] = a.s;
        }
        if (A.dx) {
            const Ref t_of(a.m, A.c);
            const float inv = 1.f / a.s;
#pragma unroll
            for (int i = 0; i < K; ++i)
                if (i < A.k)
                    Elem<TYPE>::store(A.dx + row * A.dx_row_bytes, i,
                                      live ? w * A.t * (__builtin_amdgcn_exp2f(t_of(v[i])) * inv - qk[i]) : 0.f);
        }
    }
}

// ================================================================================== 16 lanes per row, up to 256 scores
// Four rows to a wave: reductions stay inside the 16 lanes of a DPP row (rotations, so every lane has the result), and the
// instructions that a row needs whatever its length are shared by four.  Score i is in lane i % 16.  Alternatives are
// found one at a time, about 32 instructions each, so many of them are the wave kernel's (100000 x 64 bf16: 4 alternatives
// 19 us, with a wave per row 60 us; 20 alternatives 52 us and 69 us; 100000 x 200 bf16: 8 alternatives 64 us and 80 us).
constexpr int kGroupClasses = 256, kGroupEntries = 16;
inline bool group_tops(int k, int top) { return k <= 64 ? top <= 24 : top <= 8; }

template <int R> __device__ __forceinline__ uint32_t rotated(uint32_t v) {
    return __builtin_amdgcn_update_dpp(0, v, 0x120 + R, 0xf, 0xf, false);
}
template <int R> __device__ __forceinline__ float rotated(float v) { return __uint_as_float(rotated<R>(__float_as_uint(v))); }
__device__ __forceinline__ float group_sum(float v) {
    v += rotated<8>(v);
    v += rotated<4>(v);
    v += rotated<2>(v);
    return v + rotated<1>(v);
}
__device__ __forceinline__ float group_max(float v) {     // of numbers
    v = fmaxf(v, rotated<8>(v));
    v = fmaxf(v, rotated<4>(v));
    v = fmaxf(v, rotated<2>(v));
    return fmaxf(v, rotated<1>(v));
}
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
    v = max(v, rotated<8>(v));
    v = max(v, rotated<4>(v));
    v = max(v, rotated<2>(v));
    return max(v, rotated<1>(v));
}
__device__ __forceinline__ Stat group_merge(Stat a, float c) {
    const float m = group_max(a.m);
    rebase(a, m, c);
    a.s = group_sum(a.s);
    a.u = group_sum(a.u);
    return a;
}
template <int TYPE, int N>
__device__ __forceinline__ void load_group(const char* x, int k, float* v) {
    const int l = threadIdx.x & 15;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = l + 16 * j < k ? Elem<TYPE>::load(x, l + 16 * j) : -kInf;
}

template <int TYPE, int N, bool ENT>
__global__ __launch_bounds__(256) void log_probs_group_kernel(LogProbsArgs A) {
    const int l = threadIdx.x & 15;
    for (int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); row < A.n; row += (int64_t)gridDim.x * 16) {
        const char* x = A.x + row * A.row_bytes;
        const int id = id_of(A, row);
        float v[N];
        load_group<TYPE, N>(x, A.k, v);
        const float xid = id >= 0 ? Elem<TYPE>::load(x, id) : 0.f;
        Stat a = {-kInf, 0.f, 0.f};
        accumulate<N, ENT>(v, a, A.c);
        a = group_merge(a, A.c);
        if (l == 0) write_row(A, row, id, xid, a);
        if (!A.top) continue;
        uint32_t key[N], used = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) key[j] = l + 16 * j < A.k ? score_key(v[j]) : 0;
        for (int r = 0; r < A.top; ++r) {
            uint32_t best = 0, at = 0;
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (!(used >> j & 1) && key[j] > best) { best = key[j]; at = j; }
            const uint32_t highest = group_max(best);
            const uint32_t index = ~group_max(best == highest ? ~(l + 16 * at) : 0u);       // the lowest one
            if ((index & 15) == l) {
                used |= 1u << at;
                write_top(A, row, r, (uint64_t)highest << 32 | ~index, a);
            }
        }
    }
}

template <int TYPE, int N>
__global__ __launch_bounds__(256) void log_probs_grad_group_kernel(LogProbsGradArgs A) {
    const int l = threadIdx.x & 15;
    for (int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); row < A.n; row += (int64_t)gridDim.x * 16) {
        char* dx = A.dx + row * A.dx_row_bytes;
        float v[N];
        load_group<TYPE, N>(A.x + row * A.row_bytes, A.k, v);
        const float m = A.stats[2 * row], s = A.stats[2 * row + 1];
        const GradRow g = grad_row(A, row, s);
        const Ref t_of(m, A.c);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int i = l + 16 * j;
            if (i < A.k) Elem<TYPE>::store(dx, i, g.on ? grad_of(t_of(v[j]), g) + (i == g.id ? g.hit : 0.f) : 0.f);
        }
    }
}

template <int TYPE, int N>
__global__ __launch_bounds__(256) void distill_group_kernel(DistillArgs A) {
    const int l = threadIdx.x & 15;
    for (int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); row < A.n; row += (int64_t)gridDim.x * 16) {
        const char* x = A.x + row * A.row_bytes;
        char* dx = A.dx + row * A.dx_row_bytes;
        float w = A.weights ? A.weights[row] : 1.f;
        if (A.g_loss && w != 0.f) w *= A.g_loss[row];
        float v[N], lq = -kInf, q = 0.f, total = 0.f, sum = 0.f, xj = 0.f;
        int id = -1;
        bool first = false;
        Stat a = {-kInf, 0.f, 0.f};
        if (w != 0.f) {
            const int64_t raw = l < A.entries ? A.ids[row * A.entries + l] : -1;
            load_group<TYPE, N>(x, A.k, v);
            if (raw >= 0 && raw < A.k) {
                id = (int)raw;
                lq = load_any(A.teacher_type, A.teacher, row * A.entries + l);
                xj = Elem<TYPE>::load(x, id);
            }
            accumulate<N, false>(v, a, A.c);
            a = group_merge(a, A.c);
            lq = Ref(group_max(lq), A.c)(lq);
            q = id >= 0 ? __builtin_amdgcn_exp2f(lq) : 0.f;
            total = group_sum(q);
            lq -= __builtin_amdgcn_logf(total);
            q *= 1.f / total;
            // of a class named more than once the first entry stands for all
            sum = q;
            first = id >= 0;
            auto other = [&](int id2, float q2, uint32_t lane2) {
                if (id2 == id) {
                    sum += q2;
                    if (lane2 < (uint32_t)l) first = false;
                }
            };
            if (A.dx) {
#define CD_OTHER(R) other((int)rotated<R>((uint32_t)id), rotated<R>(q), rotated<R>((uint32_t)l));
                CD_OTHER(1) CD_OTHER(2) CD_OTHER(3) CD_OTHER(4) CD_OTHER(5) CD_OTHER(6) CD_OTHER(7) CD_OTHER(8)
                CD_OTHER(9) CD_OTHER(10) CD_OTHER(11) CD_OTHER(12) CD_OTHER(13) CD_OTHER(14) CD_OTHER(15)
#undef CD_OTHER
            }
        }
        const bool on = w != 0.f && total != 0.f, live = on && a.s != 0.f;
        if (A.loss) {
            const float loss = w * (A.t * A.t) * group_sum(on && id >= 0 ? loss_term(q, lq, xj, a, A.c, A.t) : 0.f);
            if (l == 0) {
                A.loss[row] = on ? loss : 0.f;
                A.stats[2 * row] = a.m;
                A.stats[2 * row + 1] = a.s;
            }
        }
        if (!A.dx) continue;
        const Ref t_of(a.m, A.c);
        const float f = live ? w * A.t / a.s : 0.f;
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (l + 16 * j < A.k)
                Elem<TYPE>::store(dx, l + 16 * j, live ? f * __builtin_amdgcn_exp2f(t_of(v[j])) : 0.f);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");          // the row first, then the teacher's classes
        if (live && first)
            Elem<TYPE>::store(dx, id, w * A.t * (__builtin_amdgcn_exp2f(t_of(xj)) * (1.f / a.s) - sum));
    }
}

// ================================================================================== one wave per row, up to 4096 scores
// The row stays in the wave's registers, no barrier, and four rows to a workgroup: 30000 x 2000 bf16 with 20 alternatives
// takes 57 us so and 152 us with a workgroup per row, 30000 x 4000 loss and gradient 92 us and 183 us.  Beyond 2048
// scores for log_probs, whose alternatives need registers of their own (it goes by the length alone, so without alternatives too),
// and beyond 8 KB for the others the registers leave too few waves.  Up to 512 scores one score at a time, score i in lane
// i % 64; above that vectors of 16 bytes, so that every lane has some, and the rest of a row one score per lane (50000 x
// 1000 bf16: 27 us with vectors, 83 us without).
constexpr int kWaveClasses = 2048, kWaveBytes = 8192;

template <int TYPE, int N> struct SpreadRow {
    static constexpr int kCount = N;                      // scores of a lane
    float v[N];
    int k;
    __device__ __forceinline__ void load(const char* x, int k_) {
        k = k_;
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = index(j) < k ? Elem<TYPE>::load(x, index(j)) : -kInf;
    }
    __device__ __forceinline__ int index(int j) const { return (threadIdx.x & 63) + 64 * j; }
    __device__ __forceinline__ bool valid(int j) const { return index(j) < k; }
    __device__ __forceinline__ float value(int j) const { return v[j]; }
    __device__ __forceinline__ void pin() {}
    template <bool ENT> __device__ __forceinline__ void add(Stat& a, float c) const { accumulate<N, ENT>(v, a, c); }
    __device__ __forceinline__ float at(int id) const {   // of a uniform id
        float r = 0.f;
#pragma unroll
        for (int j = 0; j < N; ++j) if (id >> 6 == j) r = lane_of(v[j], id & 63);
        return r;
    }
    template <class F> __device__ __forceinline__ void write(char* dx, F f) const {
#pragma unroll
        for (int j = 0; j < N; ++j) if (valid(j)) Elem<TYPE>::store(dx, index(j), f(v[j]));
    }
};
template <int TYPE, int V> struct VectorRow {
    using E = Elem<TYPE>;
    static constexpr int kCount = V * E::kVec + 1;
    u32x4 w[V];
    float single;
    const char* x;
    int k, nv;
    __device__ __forceinline__ void load(const char* x_, int k_) {
        x = x_;
        k = k_;
        nv = k / E::kVec;
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int u = 0; u < V; ++u) {
            w[u] = u32x4{E::kNegInf, E::kNegInf, E::kNegInf, E::kNegInf};
            if (lane + 64 * u < nv) w[u] = reinterpret_cast<const u32x4_any*>(x + 1024 * u)[lane];
        }
        single = nv * E::kVec + lane < k ? E::load(x, nv * E::kVec + lane) : -kInf;
    }
    __device__ __forceinline__ int index(int j) const {
        const int lane = threadIdx.x & 63;
        return j == V * E::kVec ? nv * E::kVec + lane : (lane + 64 * (j / E::kVec)) * E::kVec + j % E::kVec;
    }
    __device__ __forceinline__ bool valid(int j) const {
        return j == V * E::kVec ? index(j) < k : (int)(threadIdx.x & 63) + 64 * (j / E::kVec) < nv;
    }
    __device__ __forceinline__ float value(int j) const {
        if (j == V * E::kVec) return single;
        float xs[E::kVec];
        E::unpack(w[j / E::kVec], xs);
        return xs[j % E::kVec];
    }
    template <bool ENT> __device__ __forceinline__ void add(Stat& a, float c) const {
        constexpr int U = V < 4 ? V : 4;
#pragma unroll
        for (int u = 0; u < V; u += U) {
            float xs[U * E::kVec];
#pragma unroll
            for (int i = 0; i < U; ++i) E::unpack(w[u + i], xs + i * E::kVec);
            accumulate<U * E::kVec, ENT>(xs, a, c);
        }
        accumulate<1, ENT>(&single, a, c);
    }
    // keeps the compiler from unpacking the row outside a loop, which takes twice the registers
    __device__ __forceinline__ void pin() {
#pragma unroll
        for (int u = 0; u < V; ++u) asm volatile("" : "+v"(w[u]));
    }
    __device__ __forceinline__ float at(int id) const { return E::load(x, id); }
    template <class F> __device__ __forceinline__ void write(char* dx, F f) const {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int u = 0; u < V; ++u) {
            float d[E::kVec];
            E::unpack(w[u], d);
#pragma unroll
            for (int i = 0; i < E::kVec; ++i) d[i] = f(d[i]);
            if (lane + 64 * u < nv) reinterpret_cast<u32x4_any*>(dx + 1024 * u)[lane] = E::pack(d);
        }
        if (nv * E::kVec + lane < k) E::store(dx, nv * E::kVec + lane, f(single));
    }
};

// As block_top, from the registers; where more than 64 scores reach T (equal ones), and for NaN, the K-th largest key
// itself takes the place of T.
template <class Row, class Emit>
__device__ __forceinline__ void wave_top(Row& r, int K, float mine, bool nan, uint64_t* list, Emit emit) {
    const int lane = threadIdx.x & 63;
    const uint64_t below = (1ull << lane) - 1;
    int count = 0;
    r.pin();
    if (!nan) {
        const uint32_t high[1] = {score_key(mine)};
        const float t = key_score(kth_key<0, 1>(high, K));
#pragma unroll
        for (int j = 0; j < Row::kCount; ++j) {
            const bool take = r.value(j) >= t && r.valid(j);
            const uint64_t taken = __ballot(take);
            if (taken) {
                const int at = count + __popcll(taken & below);
                if (take && at < 64) list[at] = full_key(r.value(j), r.index(j));
                count += __popcll(taken);
            }
        }
    }
    if (nan || count > 64) {
        uint64_t t = 0;
        for (int b = 63; b >= 0; --b) {
            const uint64_t up = t | 1ull << b;
            int c = 0;
            r.pin();
#pragma unroll
            for (int j = 0; j < Row::kCount; ++j)
                c += __popcll(__ballot(r.valid(j) && full_key(r.value(j), r.index(j)) >= up));
            if (c >= K) t = up;
        }
        count = 0;
        r.pin();
#pragma unroll
        for (int j = 0; j < Row::kCount; ++j) {
            const uint64_t key = full_key(r.value(j), r.index(j));
            const bool take = r.valid(j) && key >= t;
            const uint64_t taken = __ballot(take);
            if (take) list[count + __popcll(taken & below)] = key;
            count += __popcll(taken);
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (lane < count) {
        const uint64_t mykey = list[lane];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < count; ++j) rank += list[j] > mykey;
        if (rank < K) emit(rank, mykey);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

template <class Row, bool ENT>
__global__ __launch_bounds__(256) void log_probs_wave_kernel(LogProbsArgs A) {
    __shared__ uint64_t list[4][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int64_t row = (int64_t)blockIdx.x * 4 + wave; row < A.n; row += (int64_t)gridDim.x * 4) {
        const int id = id_of(A, row);
        Row r;
        r.load(A.x + row * A.row_bytes, A.k);
        const float xid = id >= 0 ? r.at(id) : 0.f;
        Stat a = {-kInf, 0.f, 0.f};
        r.template add<ENT>(a, A.c);
        const float mine = a.m;
        a = wave_merge(a, A.c);
        if (lane == 0) write_row(A, row, id, xid, a);
        if (A.top)
            wave_top(r, A.top, mine, a.s != a.s, list[wave], [&](int rank, uint64_t key) { write_top(A, row, rank, key, a); });
    }
}

template <class Row, int TYPE>
__global__ __launch_bounds__(256) void log_probs_grad_wave_kernel(LogProbsGradArgs A) {
    const int lane = threadIdx.x & 63;
    for (int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); row < A.n;
         row += (int64_t)gridDim.x * 4) {
        char* dx = A.dx + row * A.dx_row_bytes;
        Row r;
        r.load(A.x + row * A.row_bytes, A.k);
        const float m = A.stats[2 * row], s = A.stats[2 * row + 1];
        const GradRow g = grad_row(A, row, s);
        const Ref t_of(m, A.c);
        const float hit = g.id >= 0 ? grad_of(t_of(r.at(g.id)), g) + g.hit : 0.f;
        r.write(dx, [&](float v) { return g.on ? grad_of(t_of(v), g) : 0.f; });
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");          // the row first, then its class
        if (lane == 0 && g.id >= 0) Elem<TYPE>::store(dx, g.id, hit);
    }
}

template <class Row, int TYPE, int PER>
__global__ __launch_bounds__(256) void distill_wave_kernel(DistillArgs A) {
    const int lane = threadIdx.x & 63;
    for (int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); row < A.n;
         row += (int64_t)gridDim.x * 4) {
        const char* x = A.x + row * A.row_bytes;
        char* dx = A.dx + row * A.dx_row_bytes;
        float w = A.weights ? A.weights[row] : 1.f;
        if (A.g_loss && w != 0.f) w *= A.g_loss[row];
        Row r;
        Stat a = {-kInf, 0.f, 0.f};
        Teacher<PER> te;
        te.total = 0.f;
        if (w != 0.f) {
            load_entries<PER>(te, A, row);
            r.load(x, A.k);
            share_out<PER>(te, A);
            load_student<TYPE, PER>(te, x, Part{0, A.k});
            r.template add<false>(a, A.c);
            a = wave_merge(a, A.c);
        }
        const bool on = w != 0.f && te.total != 0.f, live = on && a.s != 0.f;
        if (A.loss) {
            const float loss = on ? teacher_loss<PER>(te, a, A, w) : 0.f;
            if (lane == 0) {
                A.loss[row] = loss;
                A.stats[2 * row] = a.m;
                A.stats[2 * row + 1] = a.s;
            }
        }
        if (!A.dx) continue;
        if (live) {
            const Ref t_of(a.m, A.c);
            const float f = w * A.t / a.s;
            r.write(dx, [&](float v) { return f * __builtin_amdgcn_exp2f(t_of(v)); });
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");      // the row first, then the teacher's classes
            fix_gradient<TYPE, PER>(te, a, A, w, dx, Part{0, A.k});
        } else {
            for (int i = lane; i < A.k; i += 64) Elem<TYPE>::store(dx, i, 0.f);
        }
    }
}

constexpr int64_t kMaxGrid = 1 << 20;       // workgroups of a launch; further rows are taken by a loop
unsigned row_grid(int64_t n) { return (unsigned)std::min(n, kMaxGrid); }

int elem_size(int type) { return type == CD_T_F32 ? 4 : 2; }

// Threads of a workgroup that reads a row.  With rows enough for every CU, few threads per row: several rows then share a
// CU, and one's reads fill another's waits (20 alternatives: 30000 x 4000 bf16 98 us with 128 threads, 162 with 256, 301
// with 512; 20000 x 16000 bf16 174, 159, 209; 8000 x 64000 bf16 327, 243, 215; 4096 x 128000 bf16 263 with 256, 217 with 512, 249
// with 1024).  With few rows a row's own time counts (200 x 32000 bf16: 20 us with 128, 12.9 with 256, 10 with 512; 64 x
// 131072 bf16: 29 with 256, 19 with 512, 16 with 1024).  Where 256 threads, six workgroups to a CU, hold all rows at
// once and 512, three, would need a second round: 256 (1000 x 50021 f32: 39 us against 44; the band of 769 to 1536 rows
// follows from the numbers of workgroups that 256 CUs hold, and is measured at this size alone).
int block_threads(const RowsIn& in) {
    const int64_t bytes = (int64_t)in.k * elem_size(in.type);
    if (bytes <= 16384) return in.n >= 512 ? 128 : 256;
    if (bytes <= 65536) return in.n >= 512 ? 256 : 512;
    if (in.n <= 256) return 1024;
    return in.n > 768 && in.n <= 1536 ? 256 : 512;
}

// CALL(type, ...) for the type of the scores
#define CD_BY_TYPE(type, CALL, ...)                                     \
    do {                                                                \
        if ((type) == CD_T_F32) { CALL(CD_T_F32, __VA_ARGS__); }        \
        else if ((type) == CD_T_BF16) { CALL(CD_T_BF16, __VA_ARGS__); } \
        else { CALL(CD_T_F16, __VA_ARGS__); }                           \
    } while (0)

// CALL(type, row) for the way a wave holds a row of up to kGroupClasses scores, ...
#define CD_WAVE_ROWS_SHORT(in, CALL)                                                               \
    do {                                                                                           \
        if ((in).k <= 64) { CD_BY_TYPE((in).type, CD_SPREAD, 1, CALL); }                           \
        else { CD_BY_TYPE((in).type, CD_SPREAD, 4, CALL); }                                        \
    } while (0)
#define CD_SPREAD(TY, N, CALL) CALL(TY, SpreadRow<TY, N>)
// ... of up to kWaveClasses, ...
#define CD_WAVE_ROWS(in, CALL)                                                                     \
    do {                                                                                           \
        if ((in).k <= 512) { CD_BY_TYPE((in).type, CD_SPREAD, 8, CALL); }                          \
        else if ((in).k <= 1024) { CD_BY_TYPE((in).type, CD_VECTORS, 1, CALL); }                   \
        else { CD_BY_TYPE((in).type, CD_VECTORS, 2, CALL); }                                       \
    } while (0)
#define CD_VECTORS(TY, KILO, CALL) CALL(TY, VectorRow<TY, 16 / Elem<TY>::kVec * KILO>)
// ... and of 16-bit scores beyond that, up to kWaveBytes: for gradients and for distill's loss, not for log_probs
#define CD_WAVE_ROWS_16(in, CALL)                                                                  \
    do {                                                                                           \
        if ((in).type == CD_T_BF16) { CALL(CD_T_BF16, VectorRow<CD_T_BF16, 8>); }                  \
        else { CALL(CD_T_F16, VectorRow<CD_T_F16, 8>); }                                           \
    } while (0)
bool wave_row_16(const RowsIn& in) { return in.type != CD_T_F32 && in.k <= kWaveBytes / 2; }

unsigned thread_grid(int64_t n) { return row_grid((n + 63) / 64); }
unsigned group_grid(int64_t n) { return row_grid((n + 15) / 16); }
unsigned wave_grid(int64_t n) { return row_grid((n + 3) / 4); }
constexpr int64_t kSplitBytes = 128 << 10, kSplitRows = 64;

}  // namespace

// Workgroups per row of the calls that need a second kernel to join them: few rows, long enough that the second launch costs
// less than one CU's reading (1 x 262144 f32, loss alone: 7.5 us split, 41 us with one workgroup; 16 x 131072 bf16 with 20
// alternatives 12.3 and 14.7; 64 x 131072 bf16 15.2 and 15.7).  The limit is right for rows of that length; longer ones lose by it:
// 65 x 262144 f32 takes 24 us with a workgroup per row, 64 rows 18 us split.
static int join_parts(int64_t n, int k, int type) {
    const int64_t bytes = (int64_t)k * elem_size(type);
    if (bytes < kSplitBytes || n > kSplitRows) return 1;
    int parts = 2;
    while (parts < 64 && n * parts < 512 && bytes / parts > 32768) parts *= 2;
    return parts;
}
// ... and of the gradients, whose parts need no join: 16 workgroups per CU, of 16 KB at least (515 x 32003 f16: 17.7 us so,
// 22.7 with four per CU, 20.2 with 8 KB)
static unsigned grad_parts(int64_t n, int k, int type) {
    const int64_t bytes = (int64_t)k * elem_size(type);
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>(4096 / n, bytes / 16384));
}

size_t rows_workspace(int64_t n, int k, int type, int top) {
    const int parts = join_parts(n, k, type);
    return parts == 1 ? 0 : (size_t)n * (parts * (sizeof(float4) + top * sizeof(uint64_t)) + kMaxTeacher * sizeof(float));
}

int launch_log_probs(const RowsIn& in, const int64_t* ids, int top, float* stats, float* logp, float* entropy,
                     float* top_logp, int64_t* top_ids, void* workspace, hipStream_t s) {
    LogProbsArgs A = {static_cast<const char*>(in.x), in.n, in.stride * elem_size(in.type), in.k, top,
                      kLog2e / in.temperature, in.temperature, ids, stats, logp, entropy, top_logp, top_ids};
    A.parts = join_parts(in.n, in.k, in.type);
    A.part_stats = static_cast<float4*>(workspace);
    A.part_keys = reinterpret_cast<uint64_t*>(A.part_stats + in.n * A.parts);
    const dim3 parts((unsigned)in.n, (unsigned)A.parts);
#define SHORT(TY, K) log_probs_thread_kernel<TY, K><<<thread_grid(in.n), 64, 0, s>>>(A)
#define WAVE(TY, ...)                                                                               \
    if (entropy) log_probs_wave_kernel<__VA_ARGS__, true><<<wave_grid(in.n), 256, 0, s>>>(A);       \
    else log_probs_wave_kernel<__VA_ARGS__, false><<<wave_grid(in.n), 256, 0, s>>>(A)
#define BLOCK(TY, TH)                                                                       \
    if (entropy) log_probs_block_kernel<TY, TH, true><<<row_grid(in.n), TH, 0, s>>>(A);     \
    else log_probs_block_kernel<TY, TH, false><<<row_grid(in.n), TH, 0, s>>>(A)
#define GROUP(TY, N)                                                                                \
    if (entropy) log_probs_group_kernel<TY, N, true><<<group_grid(in.n), 256, 0, s>>>(A);           \
    else log_probs_group_kernel<TY, N, false><<<group_grid(in.n), 256, 0, s>>>(A)
#define PARTS(TY, TH)                                                                       \
    if (entropy) log_probs_part_kernel<TY, TH, true><<<parts, TH, 0, s>>>(A);               \
    else log_probs_part_kernel<TY, TH, false><<<parts, TH, 0, s>>>(A);                      \
    log_probs_join_kernel<TY><<<(unsigned)in.n, 256, 0, s>>>(A)
    if (in.k <= 4) CD_BY_TYPE(in.type, SHORT, 4);
    else if (in.k <= kThreadClasses) CD_BY_TYPE(in.type, SHORT, kThreadClasses);
    else if (in.k <= 64 && group_tops(in.k, top)) CD_BY_TYPE(in.type, GROUP, 4);
    else if (in.k <= kGroupClasses && group_tops(in.k, top)) CD_BY_TYPE(in.type, GROUP, 16);
    else if (in.k <= kGroupClasses) CD_WAVE_ROWS_SHORT(in, WAVE);
    else if (in.k <= kWaveClasses) CD_WAVE_ROWS(in, WAVE);
    else if (A.parts > 1) CD_BY_TYPE(in.type, PARTS, 512);
    else if (block_threads(in) == 128) CD_BY_TYPE(in.type, BLOCK, 128);
    else if (block_threads(in) == 256) CD_BY_TYPE(in.type, BLOCK, 256);
    else if (block_threads(in) == 512) CD_BY_TYPE(in.type, BLOCK, 512);
    else CD_BY_TYPE(in.type, BLOCK, 1024);
#undef SHORT
#undef WAVE
#undef GROUP
#undef BLOCK
#undef PARTS
    CD_HIP(hipGetLastError());
    return CD_OK;
}

int launch_log_probs_backward(const RowsIn& in, const int64_t* ids, const float* stats, const float* entropy,
                              const float* g_logp, const float* g_entropy, void* dx, int64_t dx_stride, hipStream_t s) {
    const int size = elem_size(in.type);
    const LogProbsGradArgs A = {static_cast<const char*>(in.x), static_cast<char*>(dx), in.n, in.stride * size,
                                dx_stride * size, in.k, kLog2e / in.temperature, 1.f / in.temperature, ids, stats,
                                entropy, g_logp, g_entropy};
#define SHORT(TY, K) log_probs_grad_thread_kernel<TY, K><<<thread_grid(in.n), 64, 0, s>>>(A)
#define GROUP(TY, N) log_probs_grad_group_kernel<TY, N><<<group_grid(in.n), 256, 0, s>>>(A)
#define WAVE(TY, ...) log_probs_grad_wave_kernel<__VA_ARGS__, TY><<<wave_grid(in.n), 256, 0, s>>>(A)
    const dim3 grid(row_grid(in.n), grad_parts(in.n, in.k, in.type));
#define BLOCK(TY, TH) log_probs_grad_kernel<TY, TH><<<grid, TH, 0, s>>>(A)
    if (in.k <= 4) CD_BY_TYPE(in.type, SHORT, 4);
    else if (in.k <= kThreadClasses) CD_BY_TYPE(in.type, SHORT, kThreadClasses);
    else if (in.k <= 64) CD_BY_TYPE(in.type, GROUP, 4);
    else if (in.k <= kGroupClasses) CD_BY_TYPE(in.type, GROUP, 16);
    else if (in.k <= kWaveClasses) CD_WAVE_ROWS(in, WAVE);
    else if (wave_row_16(in)) CD_WAVE_ROWS_16(in, WAVE);
    else CD_BY_TYPE(in.type, BLOCK, 256);
#undef SHORT
#undef GROUP
#undef WAVE
#undef BLOCK
    CD_HIP(hipGetLastError());
    return CD_OK;
}

static DistillArgs distill_args(const RowsIn& in, const TeacherIn& te, float* stats, float* loss, const float* g_loss,
                                void* dx, int64_t dx_stride) {
    const int size = elem_size(in.type);
    return {static_cast<const char*>(in.x), static_cast<char*>(dx), in.n, in.stride * size, dx_stride * size, in.k,
            te.entries, te.type, kLog2e / in.temperature, in.temperature, te.ids, te.scores, te.weights, g_loss, stats,
            loss};
}

// by the entries that a lane of the wave that looks after the teacher has
#define PER_LANE(ONE, TWO, FOUR)              \
    if (A.entries <= 64) { ONE; }             \
    else if (A.entries <= 128) { TWO; }       \
    else { FOUR; }

// rows that a thread or a wave takes, for which the gradient alone computes everything anew; false: longer ones
static bool launch_short_distill(const RowsIn& in, const DistillArgs& A, hipStream_t s) {
#define SHORT(TY, K) distill_thread_kernel<TY, K><<<thread_grid(in.n), 64, 0, s>>>(A)
#define GROUP(TY, N) distill_group_kernel<TY, N><<<group_grid(in.n), 256, 0, s>>>(A)
#define WAVE(TY, ...)                                                                              \
    PER_LANE((distill_wave_kernel<__VA_ARGS__, TY, 1><<<wave_grid(in.n), 256, 0, s>>>(A)),           \
             (distill_wave_kernel<__VA_ARGS__, TY, 2><<<wave_grid(in.n), 256, 0, s>>>(A)),           \
             (distill_wave_kernel<__VA_ARGS__, TY, 4><<<wave_grid(in.n), 256, 0, s>>>(A)))
    if (in.k <= 4 && A.entries <= 16) CD_BY_TYPE(in.type, SHORT, 4);
    else if (in.k <= kThreadClasses && A.entries <= 16) CD_BY_TYPE(in.type, SHORT, kThreadClasses);
    else if (in.k <= 64 && A.entries <= kGroupEntries) CD_BY_TYPE(in.type, GROUP, 4);
    else if (in.k <= kGroupClasses && A.entries <= kGroupEntries) CD_BY_TYPE(in.type, GROUP, 16);
    else if (in.k <= kGroupClasses) CD_WAVE_ROWS_SHORT(in, WAVE);
    else if (in.k <= kWaveClasses) CD_WAVE_ROWS(in, WAVE);
    else if (wave_row_16(in)) CD_WAVE_ROWS_16(in, WAVE);
    else return false;
#undef SHORT
#undef GROUP
#undef WAVE
    return true;
}

int launch_distill(const RowsIn& in, const TeacherIn& te, float* stats, float* loss, void* dx, int64_t dx_stride,
                   void* workspace, hipStream_t s) {
    DistillArgs A = distill_args(in, te, stats, loss, nullptr, dx, dx_stride);
    A.parts = join_parts(in.n, in.k, in.type);
    A.part_stats = static_cast<float4*>(workspace);
    A.part_x = reinterpret_cast<float*>(A.part_stats + in.n * A.parts);
    const dim3 parts((unsigned)in.n, (unsigned)A.parts), writers((unsigned)in.n, dx ? grad_parts(in.n, in.k, in.type) : 1);
    if (!launch_short_distill(in, A, s)) {
#define PARTS(TY, TH)                                                                                       \
    distill_part_kernel<TY, TH><<<parts, TH, 0, s>>>(A);                                                    \
    PER_LANE((distill_join_kernel<TY, 256, 1><<<writers, 256, 0, s>>>(A)),                                    \
             (distill_join_kernel<TY, 256, 2><<<writers, 256, 0, s>>>(A)),                                    \
             (distill_join_kernel<TY, 256, 4><<<writers, 256, 0, s>>>(A)))
#define BLOCK(TY, TH)                                                                                       \
    PER_LANE((distill_block_kernel<TY, TH, 1><<<row_grid(in.n), TH, 0, s>>>(A)),                              \
             (distill_block_kernel<TY, TH, 2><<<row_grid(in.n), TH, 0, s>>>(A)),                              \
             (distill_block_kernel<TY, TH, 4><<<row_grid(in.n), TH, 0, s>>>(A)))
#define HELD(TY, TH, V)                                                                                     \
    PER_LANE((distill_held_kernel<TY, TH, V, 1><<<row_grid(in.n), TH, 0, s>>>(A)),                          \
             (distill_held_kernel<TY, TH, V, 2><<<row_grid(in.n), TH, 0, s>>>(A)),                          \
             (distill_held_kernel<TY, TH, V, 4><<<row_grid(in.n), TH, 0, s>>>(A)))
        const int vectors = in.k / (16 / elem_size(in.type));
        if (A.parts > 1) CD_BY_TYPE(in.type, PARTS, 512);
        else if (dx && vectors <= 256 * 8) CD_BY_TYPE(in.type, HELD, 256, 8);
        else if (dx && vectors <= 512 * 8) CD_BY_TYPE(in.type, HELD, 512, 8);
        else if (dx && vectors <= 512 * 16) CD_BY_TYPE(in.type, HELD, 512, 16);
        else if (dx && vectors <= 1024 * 16) CD_BY_TYPE(in.type, HELD, 1024, 16);
        else if (block_threads(in) == 128) CD_BY_TYPE(in.type, BLOCK, 128);
        else if (block_threads(in) == 256) CD_BY_TYPE(in.type, BLOCK, 256);
        else if (block_threads(in) == 512) CD_BY_TYPE(in.type, BLOCK, 512);
        else CD_BY_TYPE(in.type, BLOCK, 1024);
#undef BLOCK
#undef HELD
#undef PARTS
    }
    CD_HIP(hipGetLastError());
    return CD_OK;
}

int launch_distill_backward(const RowsIn& in, const TeacherIn& te, const float* stats, const float* g_loss, void* dx,
                            int64_t dx_stride, hipStream_t s) {
    DistillArgs A = distill_args(in, te, nullptr, nullptr, g_loss, dx, dx_stride);
    if (!launch_short_distill(in, A, s)) {
        A.stats = const_cast<float*>(stats);              // only read
        const dim3 grid(row_grid(in.n), grad_parts(in.n, in.k, in.type));
#define BLOCK(TY, TH)                                                                                       \
    PER_LANE((distill_grad_kernel<TY, TH, 1><<<grid, TH, 0, s>>>(A)),                                         \
             (distill_grad_kernel<TY, TH, 2><<<grid, TH, 0, s>>>(A)),                                         \
             (distill_grad_kernel<TY, TH, 4><<<grid, TH, 0, s>>>(A)))
        CD_BY_TYPE(in.type, BLOCK, 256);
#undef BLOCK
    }
    CD_HIP(hipGetLastError());
    return CD_OK;
}

}  // namespace cd
