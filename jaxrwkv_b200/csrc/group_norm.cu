// Group norm of rows of C channels, statistics per row and group of D = C / G consecutive channels, with an activation and,
// where a gate is given, a product with the activated gate (the output stage of RWKV-5, 5.2 and 6 has silu there):
//   xh = (x - mean) / sqrt(var + eps)   n = xh weight + bias   y = act(n), or n act(gate)
// Backward, dn = gy act'(n) or gy act(gate):
//   dgate = gy n act'(gate)   dxh = dn weight   dx = rstd (dxh - mean(dxh) - xh mean(dxh xh))
//   dweight = sum over rows of dn xh   dbias = sum over rows of dn
// The statistics are computed again in the backward (its x is read anyway), so nothing is kept.
//
// One pass over the rows, bound by memory: 3 elements a channel forward, 5 backward (2 and 3 without a gate).  A team of threads owns one group: lanes
// of a warp with one or two 16-byte pieces of the row each (up to eight pairs where 16 bytes do not fit), or a whole
// CTA where the group is wider than that.  The row's values stay in registers from the mean over the centred squares to the
// result.  A team keeps its group from row to row, so that weight and bias are read once and their gradients are added up in
// registers; they leave as partial rows, which a second kernel adds in a fixed order.
// 32768 rows of 32 groups of 64 channels, bf16, silu of a gate: forward 60 us, 1.04 of the measured copy rate; backward 110 us, 0.94, and
// 4 us for the sums behind it (ncu's clock; between events around a call whose operands are not in L2, as the figures below, 74 and 125 in all).
// Groups that are no power of two of pieces leave lanes idle (24 groups of 72: 5 of 32) and take longer sums: 20 groups of 80 reach 0.70 and
// 0.69 of the copy rate, 32 of 40 0.64 and 0.71.  Single elements, as of 32 groups of 61, reach 0.40 and 0.39, bound by the number of loads.
// Backward of wide groups: 8 of 512 0.66 gated and 0.48 not, one of 2048 0.49 and 0.31 (eight warps an SM, one row ahead, in whole CTAs
// four barriers a row), one of 5120 0.27 and one of 4097 0.06 (the registers of 16 channels a thread spill).
#include <initializer_list>
#include <type_traits>

#include "common.cuh"
#include "device_once.cuh"
#include "gate_math.cuh"
#include "host_calls.h"
#include "tc05.cuh"

namespace b200wkv {
namespace {

constexpr int kChain = 16;                 // rows that a thread adds up in registers
constexpr int kMaxPartials = 1024;         // partial rows of the parameters' gradients
constexpr int kMaxThreads = 512;

struct Params {                            // weight or bias; p NULL: ones or zeros
    const void* p;
    int f32;
    __device__ __forceinline__ float at(int c) const { return f32 ? ((const float*)p)[c] : __bfloat162float(((const __nv_bfloat16*)p)[c]); }
    // N from the c-th on as pairs, of which the first `valid` are there; 16-byte loads where `vectors`
    template <int N> __device__ __forceinline__ void load(int c, int valid, bool vectors, float otherwise, F2* to) const {
        if (p == nullptr) {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) to[i] = both(otherwise);
        } else if (N % 4 == 0 && vectors) {
            if (f32) {
#pragma unroll
                for (int i = 0; i < N / 4; ++i) {
                    const ulonglong2 q = ((const ulonglong2*)((const float*)p + c))[i];
                    to[2 * i].v = q.x;
                    to[2 * i + 1].v = q.y;
                }
            } else {
#pragma unroll
                for (int i = 0; i < N / 4; ++i) {
                    const uint2 q = ((const uint2*)((const __nv_bfloat16*)p + c))[i];
                    to[2 * i] = unpack_pair(q.x);
                    to[2 * i + 1] = unpack_pair(q.y);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) to[i] = make_f2(at(c + 2 * i), 2 * i + 1 < valid ? at(c + 2 * i + 1) : 0.f);
        }
    }
};
struct Problem {
    long long rows;
    int C, G, D, act;
    float eps;
    const void *x, *gate;
    long long x_stride, gate_stride;       // elements from row to row
    Params weight, bias;
    int team;                              // threads of a team
    int per_cta;                           // teams at work in a CTA: all of them, or a multiple of G
    int parallel;                          // rows at a time over the grid
    int param_vectors;                     // weight and bias begin on 16 bytes
    int totals;                            // where the threads' sums beyond kChain rows begin in shared memory; -1: nobody takes so many
    int reduce;                            // teams of one group within a CTA are added up (per_cta is a multiple of G)
};

// A piece of a row as it lies in memory: VEC adjacent elements of one load, or (kWhole false) two of one load each, of which the second may
// lie behind the group's end and is 0 then.
template <typename T, int VEC, bool kWhole> struct Piece {
    static constexpr int kWords = VEC * (int)sizeof(T) / 4;
    uint32_t q[kWords];
    __device__ __forceinline__ void load(const T* p, bool) {
        if constexpr (kWords == 4) {
            const uint4 v = *(const uint4*)p;
            q[0] = v.x; q[1] = v.y; q[2] = v.z; q[3] = v.w;
        } else if constexpr (kWords == 2) {
            const uint2 v = *(const uint2*)p;
            q[0] = v.x; q[1] = v.y;
        } else q[0] = *(const uint32_t*)p;
    }
    __device__ __forceinline__ void unpack(F2* v) const {
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i)
            v[i] = sizeof(T) == 4 ? make_f2(__uint_as_float(q[2 * i % kWords]), __uint_as_float(q[(2 * i + 1) % kWords])) : unpack_pair(q[i % kWords]);
    }
    __device__ __forceinline__ static void store(T* p, const F2* v, bool) {
        uint32_t w[kWords];
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
            const float2 t = parts(v[i]);
            if constexpr (sizeof(T) == 4) {
                w[2 * i] = __float_as_uint(t.x);
                w[2 * i + 1] = __float_as_uint(t.y);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(t.x, t.y);
                w[i] = *(const uint32_t*)&h;
            }
        }
        if constexpr (kWords == 4) *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]);
        else if constexpr (kWords == 2) *(uint2*)p = make_uint2(w[0], w[1]);
        else *(uint32_t*)p = w[0];
    }
};
template <typename T, int VEC> struct Piece<T, VEC, false> {
    static_assert(VEC == 2, "two elements");
    T q[2];
    __device__ __forceinline__ void load(const T* p, bool second) {
        q[0] = p[0];
        if (second) q[1] = p[1];
    }
    __device__ __forceinline__ void unpack(F2* v) const { v[0] = make_f2(to_f32(q[0]), to_f32(q[1])); }
    __device__ __forceinline__ static void store(T* p, const F2* v, bool second) {
        const float2 t = parts(v[0]);
        p[0] = from_f32<T>(t.x);
        if (second) p[1] = from_f32<T>(t.y);
    }
};
__device__ __forceinline__ float sum_of(F2 v) {
    const float2 t = parts(v);
    return t.x + t.y;
}
__device__ __forceinline__ F2 first_alone(F2 v) { return make_f2(parts(v).x, 0.f); }

// act(z), and its derivative where it is asked for.  Below -87 silu is what it is there, -1.5e-36: sigmoid's least value, 2^-126, times the z of a
// closed gate, which may be the type's lowest number, is none of the function's values (-4).  -inf counts as closed too.
template <typename T, int kAct> __device__ __forceinline__ void activate(F2 z, F2& p, F2& dp) {
    if (kAct == B200WKV_ACT_NONE) { p = z; dp = both(1.f); return; }
    F2 s, r;
    if (kAct == B200WKV_ACT_SIGMOID) {
        sigmoid_pair<T>(z, s, r);
        p = s;
        dp = mul2(s, r);
    } else {
        const float2 t = parts(z);
        z = make_f2(max_nan(t.x, -87.f), max_nan(t.y, -87.f));
        sigmoid_pair<T, true>(z, s, r);
        p = mul2(z, s);
        dp = mul2(s, fma2(z, r, both(1.f)));
    }
}

// Where a thread's team works: group g, rows first, first + parallel, ...; none of them where `at_work` is false.  A warp has as many teams as fit
// it, and the lanes behind them are idle.
struct Place {
    int team, g, lane;
    int slot;                              // teams' lanes in a row; -1: idle
    long long first;
    bool at_work;
    __device__ __forceinline__ Place(const Problem& p, int team_) : team(team_) {
        const int per_warp = 32 / team, in_warp = (int)(threadIdx.x & 31) / team;      // (0 and 0 for whole CTAs)
        const int in_cta = team > 32 ? 0 : (int)(threadIdx.x / 32) * per_warp + in_warp, q = blockIdx.x * p.per_cta + in_cta;
        lane = team > 32 ? (int)threadIdx.x : (int)(threadIdx.x & 31) - in_warp * team;
        slot = team > 32 || in_warp < per_warp ? in_cta * team + lane : -1;
        g = q % p.G;
        first = q / p.G;
        at_work = slot >= 0 && in_cta < p.per_cta && first < p.parallel;
    }
};

// sum over the team, the same in every thread of it.  Whole CTAs: a row's sums have places of their own in `room`, so that one barrier
// each is enough (a place is written again behind the barrier of the next sum, which everyone reaches after reading it).
// kTeam: the team's lanes where they are known to the compiler, 0 for any power of two (five branches a sum), kAnyTeam for others.
constexpr int kAnyTeam = -1;
template <bool kBlock, int kTeam> __device__ __forceinline__ float team_sum(float a, const Place& at, float* room) {
    if (kTeam == kAnyTeam) {               // the first lane's is the team's
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            if (o >= at.team) break;
            const float next = __shfl_down_sync(0xffffffffu, a, o);
            if (at.lane + o < at.team) a += next;
        }
        return __shfl_sync(0xffffffffu, a, (int)(threadIdx.x & 31) - at.lane);
    }
#pragma unroll
    for (int o = 16; o > 0; o /= 2)
        if (kBlock || (kTeam > 0 ? kTeam : at.team) > o) a += __shfl_xor_sync(0xffffffffu, a, o);
    if (kBlock) {
        const int warps = blockDim.x / 32;
        if (threadIdx.x % 32 == 0) room[threadIdx.x / 32] = a;
        __syncthreads();
        a = 0.f;
        for (int w = 0; w < warps; ++w) a += room[w];
    }
    return a;
}

// The pieces of one thread: K, `step` channels apart.  kWhole false: the group's last element may be the first of a pair (`odd`).
template <typename T, int VEC, int K, bool kWhole> struct Lane {
    static constexpr int kPairs = VEC / 2;
    typedef Piece<T, VEC, kWhole> P;
    int c, step;                           // the first piece's channel in the row
    bool there[K], second[K];              // the piece; its second element (kWhole false)
    F2 w[K][kPairs], b[K][kPairs];
    __device__ __forceinline__ Lane(const Problem& p, const Place& at) : c(at.g * p.D + at.lane * VEC), step(at.team * VEC) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int d = (at.lane + k * at.team) * VEC;
            there[k] = at.at_work && d < p.D;
            second[k] = kWhole || d + 1 < p.D;
#pragma unroll
            for (int i = 0; i < kPairs; ++i) w[k][i] = b[k][i] = both(0.f);
            if (there[k]) {
                p.weight.load<VEC>(c + k * step, p.D - d, p.param_vectors, 1.f, w[k]);
                p.bias.load<VEC>(c + k * step, p.D - d, p.param_vectors, 0.f, b[k]);
            }
        }
    }
    __device__ __forceinline__ void store(T* row, int k, const F2* v) const { P::store(row + k * step, v, second[k]); }
    // x less its mean over the team (0 where there is nothing), and 1 / sqrt(var + eps)
    template <bool kBlock, int kTeam> __device__ __forceinline__ float centre(F2 (&x)[K][kPairs], const Problem& p, const Place& at, float inv_d, float* room) const {
        F2 sums = both(0.f);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int j = 0; j < kPairs; ++j) sums = add2(sums, x[k][j]);
        const F2 less = both(-team_sum<kBlock, kTeam>(sum_of(sums), at, room) * inv_d);
        sums = both(0.f);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            F2 squares = both(0.f);
#pragma unroll
            for (int j = 0; j < kPairs; ++j) {
                x[k][j] = add2(x[k][j], less);
                if (!kWhole && !second[k]) x[k][j] = first_alone(x[k][j]);
                squares = fma2(x[k][j], x[k][j], squares);
            }
            if (there[k]) sums = add2(sums, squares);
        }
        return rsqrtf(team_sum<kBlock, kTeam>(sum_of(sums), at, room + kMaxThreads / 32) * inv_d + p.eps);
    }
};
// A stream's pieces of the rows to come.  kAsync: pieces of 16 bytes travel to shared memory by cp.async, three rows in front of the one at
// work (two of two pieces each); the registers would hold one row, a third of what keeps the memory busy.  A thread reads only
// what it has asked for itself, so no barrier is needed.  Else one row ahead, in registers.
template <typename T, int VEC, int K, bool kWhole, bool kAsync> struct Rows {
    typedef Lane<T, VEC, K, kWhole> L;
    static constexpr int kAhead = !kAsync ? 1 : K == 1 ? 3 : 2;
    static constexpr size_t kBytes = kAsync ? (size_t)kAhead * K * 16 : 0;     // a thread's of shared memory
    const T* from;                         // the thread's first piece of the row to ask for next
    long long step;                        // elements to the row after it
    unsigned char* room;
    typename L::P q[K];
    __device__ __forceinline__ Rows(const void* p, long long stride, const Problem& pr, const Place& at, const L& my, int which, unsigned char* shared)
        : from((const T*)p + at.first * stride + my.c), step(pr.parallel * stride), room(shared + ((size_t)which * kAhead * K * blockDim.x + threadIdx.x) * 16), q{} {}
    __device__ __forceinline__ unsigned char* slot(int place, int k) const { return room + (size_t)(place * K + k) * blockDim.x * 16; }
    __device__ __forceinline__ void ask(int place, bool on, const L& my) {
        if (on) {
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (my.there[k]) {
                    if constexpr (kAsync) tc::cp_async16(slot(place, k), from + k * my.step, true);
                    else q[k].load(from + k * my.step, my.second[k]);
                }
        }
        from += step;
    }
    __device__ __forceinline__ void take(int place, F2 (&v)[K][L::kPairs], const L& my) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if constexpr (kAsync) {
                q[k] = typename L::P{};
                if (my.there[k]) q[k].load((const T*)slot(place, k), true);
            }
            q[k].unpack(v[k]);
        }
    }
};
// Where that pays.  32768 rows of 32 groups of 64, bf16, gated: forward 80 -> 76 us, backward 136 -> 122; 8190 rows of 8 groups of 512 (two pieces
// a thread): forward 51 -> 47, backward 79 -> 83 without a gate, 87 -> 87 with one; in fp32, where a piece is half as many numbers for the same
// instructions, backward 115 -> 134; whole CTAs a group: forward 51 -> 53, backward 103 -> 108.
template <typename T, int K, bool kWhole, bool kBlock, bool kForward> constexpr bool kAsyncRows = sizeof(T) == 2 && kWhole && !kBlock && (kForward || K == 1);

// the row at work has arrived; those behind it may be on their way
template <int kAhead, bool kAsync> __device__ __forceinline__ void asked() {
    if constexpr (kAsync) asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int kAhead, bool kAsync> __device__ __forceinline__ void arrived() {
    if constexpr (kAsync) asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
}

// A thread's sums of the parameters' gradients beyond kChain rows, in shared memory: 32768 rows are 111 a thread, and one chain of 32-bit additions
// over them is three times as far off as the terms are.  kExact: with what each addition rounds away, which the next one makes up for (Kahan's
// sum); else without, where the registers of a whole CTA have spilled and want the L1 cache (5120 channels: a pass 329 us, with 392).  dweight and
// dbias of 32768 rows of 32 groups of 64, bf16 streams: 1.1e-7 and 1.0e-7 off (2-norm) instead of 2.2e-7, the terms alone are 0.8e-7 and 0.5e-7;
// with 8 rows at a time 1.0e-7 and 0.9e-7, and 2 us more.  The pass through autograd 187 -> 185 us, without a gate 144 -> 153,
// 8192 rows of 5120 channels 317 -> 329, 16384 rows of 2048 148 -> 154, fp32 rows of 2 groups of 1000 246 -> 241, others within 3 %.
template <int kPairs, bool kExact, int kThreads> struct Totals {
    struct alignas(kExact ? 16 : 8) Sum { F2 v[kExact ? 2 : 1]; };       // the sum, and what it is too large by
    Sum* at;
    bool on;
    __device__ __forceinline__ Totals(unsigned char* shared, int from) : at((Sum*)(shared + from) + threadIdx.x), on(from >= 0) {}
    __device__ __forceinline__ static int apart() { return kThreads > 0 ? kThreads : blockDim.x; }
    __device__ __forceinline__ static F2 less(F2 a, F2 b) { return fma2(b, both(-1.f), a); }
    // (an infinite sum stays one)
    __device__ __forceinline__ static F2 of_finite(F2 s, F2 v) {
        const float2 a = parts(s), b = parts(v);
        return make_f2(isfinite(a.x) ? b.x : 0.f, isfinite(a.y) ? b.y : 0.f);
    }
    __device__ __forceinline__ static F2& of(F2* dw, F2* db, int i) { return i < kPairs ? dw[i] : db[i - kPairs]; }
    // what the registers hold, which begin anew
    __device__ __forceinline__ void add(F2* dw, F2* db, bool first) {
#pragma unroll
        for (int i = 0; i < 2 * kPairs; ++i) {
            F2& v = of(dw, db, i);
            Sum t = {};
            if (!first) t = at[i * apart()];
            if constexpr (kExact) {
                const F2 y = less(v, t.v[1]), s = add2(t.v[0], y);
                t = {{s, of_finite(s, less(less(s, t.v[0]), y))}};
            } else {
                t.v[0] = add2(t.v[0], v);
            }
            at[i * apart()] = t;
            v = both(0.f);
        }
    }
    // all of it, in the registers
    __device__ __forceinline__ void take(F2* dw, F2* db) const {
#pragma unroll
        for (int i = 0; i < 2 * kPairs; ++i) {
            F2& v = of(dw, db, i);
            const Sum t = at[i * apart()];
            if constexpr (kExact) v = less(v, t.v[1]);
            v = add2(t.v[0], v);
        }
    }
};

template <int kPairs, bool kExact> constexpr size_t kTotalBytes = 2 * kPairs * (kExact ? 16 : 8);      // a thread's

template <typename Go> __device__ __forceinline__ void by_activation(int act, Go go) {
    if (act == B200WKV_ACT_SILU) go(std::integral_constant<int, B200WKV_ACT_SILU>());
    else if (act == B200WKV_ACT_SIGMOID) go(std::integral_constant<int, B200WKV_ACT_SIGMOID>());
    else go(std::integral_constant<int, B200WKV_ACT_NONE>());
}

// CTAs of 256 threads an SM for the registers of a kernel: weight, bias, a row's values and the next row's as they lie in memory (`bytes`; a
// register for each where they are loaded one by one)
constexpr int fwd_ctas(int elements, int bytes, bool gate) { return elements <= 4 || (elements <= 8 && bytes <= 16) ? 4 : elements <= 8 || (!gate && bytes <= 32) ? 3 : 2; }
__host__ __device__ constexpr int bwd_ctas(int elements, int bytes, bool gate) { return elements <= 4 ? 3 : elements <= 8 || (!gate && bytes <= 32) ? 2 : 1; }

template <typename T, int VEC, int K, bool kWhole, bool kBlock, int kTeam, bool kGate>
__global__ void __launch_bounds__(kBlock ? kMaxThreads : 256, kBlock && VEC * K <= 8 ? 2 : kBlock ? 1 : fwd_ctas(VEC * K, VEC * K * (kWhole ? (int)sizeof(T) : 4), kGate))
group_norm_fwd_kernel(const Problem p, T* __restrict__ y) {
    typedef Lane<T, VEC, K, kWhole> L;
    __shared__ float room[kBlock ? 4 * kMaxThreads / 32 : 1];
    const Place at(p, kBlock ? (int)blockDim.x : kTeam > 0 ? kTeam : p.team);
    const L my(p, at);
    const float inv_d = 1.f / (float)p.D;
    extern __shared__ __align__(16) unsigned char shared[];
    constexpr bool kAsync = VEC == 8 && kAsyncRows<T, K, kWhole, kBlock, true>;
    typedef Rows<T, VEC, K, kWhole, kAsync> R;
    R rx(p.x, p.x_stride, p, at, my, 0, shared), rg(p.gate, p.gate_stride, p, at, my, 1, shared);
    const auto ask = [&](int place, long long row) {
        rx.ask(place, row < p.rows, my);
        if (kGate) rg.ask(place, row < p.rows, my);
        asked<R::kAhead, kAsync>();
    };
    for (int i = 0; i < R::kAhead; ++i) ask(i, at.first + (long long)i * p.parallel);
    T* py = y + at.first * p.C + my.c;
    // (teams without work go along: the sums take whole warps and CTAs)
    const long long steps = (p.rows + p.parallel - 1) / p.parallel;
    long long row = at.first;
    int place = 0;
    for (long long i = 0; i < steps; ++i, row += p.parallel, py += (long long)p.parallel * p.C) {
        F2 x[K][L::kPairs], g[K][L::kPairs];
        arrived<R::kAhead, kAsync>();
        rx.take(place, x, my);
        if (kGate) rg.take(place, g, my);
        ask(place, row + (long long)R::kAhead * p.parallel);
        place = place + 1 == R::kAhead ? 0 : place + 1;
        const F2 rstd = both(my.template centre<kBlock, kTeam>(x, p, at, inv_d, room));
        by_activation(p.act, [&](auto act) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (!my.there[k] || row >= p.rows) continue;
                F2 out[L::kPairs];
#pragma unroll
                for (int j = 0; j < L::kPairs; ++j) {
                    const F2 n = fma2(mul2(x[k][j], rstd), my.w[k][j], my.b[k][j]);
                    F2 a, da;
                    activate<T, act.value>(kGate ? g[k][j] : n, a, da);
                    out[j] = kGate ? mul2(n, a) : a;
                }
                my.store(py, k, out);
            }
        });
    }
}

template <typename T, int VEC, int K, bool kWhole, bool kBlock, int kTeam, bool kGate>
__global__ void __launch_bounds__(kBlock ? kMaxThreads : 256, kBlock ? 1 : bwd_ctas(VEC * K, VEC * K * (kWhole ? (int)sizeof(T) : 4), kGate))
group_norm_bwd_kernel(const Problem p, const T* __restrict__ gy, T* __restrict__ dx, T* __restrict__ dgate, float* __restrict__ partial) {
    typedef Lane<T, VEC, K, kWhole> L;
    constexpr int kPairs = L::kPairs;
    __shared__ float room[kBlock ? 4 * kMaxThreads / 32 : 1];
    const Place at(p, kBlock ? (int)blockDim.x : kTeam > 0 ? kTeam : p.team);
    const L my(p, at);
    const float inv_d = 1.f / (float)p.D;
    F2 dw[K][kPairs], db[K][kPairs];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < kPairs; ++i) dw[k][i] = db[k][i] = both(0.f);
    extern __shared__ __align__(16) unsigned char shared[];
    constexpr bool kAsync = VEC == 8 && kAsyncRows<T, K, kWhole, kBlock, false>;
    typedef Rows<T, VEC, K, kWhole, kAsync> R;
    const long long steps = (p.rows + p.parallel - 1) / p.parallel;
    typedef Totals<K * kPairs, !(kBlock && K * kPairs > 4), kBlock ? 0 : 256> Sums;
    Sums totals(shared, p.totals);
    R rx(p.x, p.x_stride, p, at, my, 0, shared), rd(gy, p.C, p, at, my, 1, shared), rg(p.gate, p.gate_stride, p, at, my, 2, shared);
    const auto ask = [&](int place, long long row) {
        rx.ask(place, row < p.rows, my);
        rd.ask(place, row < p.rows, my);
        if (kGate) rg.ask(place, row < p.rows, my);
        asked<R::kAhead, kAsync>();
    };
    for (int i = 0; i < R::kAhead; ++i) ask(i, at.first + (long long)i * p.parallel);
    long long dense = at.first * p.C + my.c;
    long long row = at.first;
    int place = 0;
    for (long long begin = 0; begin < steps; begin += kChain) {
        if (totals.on && begin > 0) totals.add(&dw[0][0], &db[0][0], begin == kChain);
        const int n = (int)(steps - begin < kChain ? steps - begin : kChain);
        for (int i = 0; i < n; ++i, row += p.parallel, dense += (long long)p.parallel * p.C) {
            const bool on = row < p.rows;
            F2 x[K][kPairs], g[K][kPairs], d[K][kPairs];
            arrived<R::kAhead, kAsync>();
            rx.take(place, x, my);
            rd.take(place, d, my);
            if (kGate) rg.take(place, g, my);
            ask(place, row + (long long)R::kAhead * p.parallel);
            place = place + 1 == R::kAhead ? 0 : place + 1;
            const F2 rstd = both(my.template centre<kBlock, kTeam>(x, p, at, inv_d, room));
            F2 s1 = both(0.f), s2 = both(0.f);                // of dxh and dxh xh
            by_activation(p.act, [&](auto act) {
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (!my.there[k] || !on) continue;
#pragma unroll
                    for (int j = 0; j < kPairs; ++j) {
                        const F2 xh = mul2(x[k][j], rstd), n = fma2(xh, my.w[k][j], my.b[k][j]);
                        F2 a, da;
                        activate<T, act.value>(kGate ? g[k][j] : n, a, da);
                        F2 dn = mul2(d[k][j], kGate ? a : da);
                        if (kGate) g[k][j] = mul2(mul2(d[k][j], n), da);
                        if (!kWhole && !my.second[k]) dn = first_alone(dn);
                        dw[k][j] = fma2(dn, xh, dw[k][j]);
                        db[k][j] = add2(db[k][j], dn);
                        const F2 dxh = mul2(dn, my.w[k][j]);
                        s1 = add2(s1, dxh);
                        s2 = fma2(dxh, xh, s2);
                        x[k][j] = xh;
                        d[k][j] = dxh;
                    }
                }
            });
            const F2 m1 = both(-team_sum<kBlock, kTeam>(sum_of(s1), at, room + 2 * kMaxThreads / 32) * inv_d);
            const F2 m2 = both(-team_sum<kBlock, kTeam>(sum_of(s2), at, room + 3 * kMaxThreads / 32) * inv_d);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (!my.there[k] || !on) continue;
                if (kGate) my.store(dgate + dense, k, g[k]);
#pragma unroll
                for (int j = 0; j < kPairs; ++j) d[k][j] = mul2(fma2(x[k][j], m2, add2(d[k][j], m1)), rstd);
                my.store(dx + dense, k, d[k]);
            }
        }
    }
    if (partial == nullptr) return;
    if (totals.on) totals.take(&dw[0][0], &db[0][0]);
    // partial rows (parallel or one per CTA, 2, C): weight, bias
    const auto of = [](const F2* v, int i) { return i % 2 == 0 ? parts(v[i / 2]).x : parts(v[i / 2]).y; };
    if (!kBlock && p.reduce) {             // teams of one group within the CTA are added first, a column a thread
        float* const both_sums = (float*)shared;             // (every copy into it has arrived)
#pragma unroll
        for (int k = 0; k < K; ++k) {
            __syncthreads();
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                if (at.slot < 0) continue;
                both_sums[at.slot * VEC + v] = of(dw[k], v);
                both_sums[(256 + at.slot) * VEC + v] = of(db[k], v);
            }
            __syncthreads();
            const int width = p.team * VEC, columns = 2 * p.G * width;         // of this k
            for (int t = threadIdx.x; t < columns; t += 256) {
                const int which = t / (p.G * width), g = t % (p.G * width) / width, d = t % width, c = d + k * width;
                if (c >= p.D) continue;
                double sum = 0.;
                for (int j = g; j < p.per_cta; j += p.G) sum += both_sums[which * 256 * VEC + j * width + d];
                partial[((size_t)blockIdx.x * 2 + which) * p.C + g * p.D + c] = (float)sum;
            }
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (my.there[k]) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                if (v == 1 && !my.second[k]) continue;
                partial[((size_t)at.first * 2) * p.C + my.c + k * my.step + v] = of(dw[k], v);
                partial[((size_t)at.first * 2 + 1) * p.C + my.c + k * my.step + v] = of(db[k], v);
            }
        }
}

// The partial rows' sums, in 64 bits and rounded to the parameters' type: a CTA owns 32 of the 2 C columns, its warps every sixteenth row, added in a fixed order.
__global__ void __launch_bounds__(512) group_norm_sums_kernel(const float* partial, int rows, int C, int f32, void* dweight, void* dbias) {
    __shared__ double part[16][32];
    wait_for_grid_in_front();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    double s[8] = {};
    if (c < 2 * C)
        for (int r = warp; r < rows; r += 128)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (r + 16 * j < rows) s[j] += partial[(size_t)(r + 16 * j) * 2 * C + c];
    part[warp][lane] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    __syncthreads();
    if (warp != 0 || c >= 2 * C) return;
    double t = 0.;
#pragma unroll
    for (int w = 0; w < 16; ++w) t += part[w][lane];
    void* const to = c < C ? dweight : dbias;
    if (to == nullptr) return;
    const int at = c < C ? c : c - C;
    if (f32) ((float*)to)[at] = (float)t;
    else ((__nv_bfloat16*)to)[at] = __double2bfloat16(t);
}

// How a call is cut.  Pieces of 16 bytes where rows and groups fit them, else pairs; a team as narrow as covers the group with K pieces a
// thread, which keeps the shuffles few; a whole CTA where the group is wider than a warp with K.
struct Plan {
    int vec, k, block, grid;
    bool whole;
};
// `aligned`: bytes that every row and pointer begins on.
Plan plan_of(Problem& p, int element, int aligned, bool forward) {
    Plan q;
    const int wide = 16 / element;
    q.vec = aligned >= 16 && p.D % wide == 0 ? wide : 2;
    q.whole = q.vec == wide || (aligned >= 2 * element && p.D % 2 == 0);
    const int pieces = (p.D + q.vec - 1) / q.vec;
    if (q.vec == wide) q.k = pieces <= 32 ? 1 : 2;
    else q.k = pieces <= 128 ? 4 : 8;      // bf16, 32768 rows of 4 groups of 333: forward / backward 223 / 282 us with CTAs of 64 and four pairs, 107 / 240 so
    if (pieces <= 32 * q.k) {
        q.block = 256;
        const int lanes = (pieces + q.k - 1) / q.k;
        p.team = 1;
        while (p.team < lanes) p.team *= 2;
        if (32 / lanes > 32 / p.team) p.team = lanes;    // bf16, 20 groups of 80, gated: 72 / 140 -> 67 / 116 us; 24 of 72: 86 / 163 -> 74 / 133; 32 of 48: 61 / 110 and 67 / 106
    } else {
        if (q.vec == wide) q.k = pieces <= kMaxThreads ? 1 : pieces <= 2 * kMaxThreads ? 2 : 4;
        else q.k = pieces <= 4 * kMaxThreads ? 4 : 8;
        q.block = ((pieces + q.k - 1) / q.k + 31) / 32 * 32;
        p.team = q.block;
    }
    const int teams = p.team > 32 ? 1 : q.block / 32 * (32 / p.team);
    p.reduce = p.G * 4 <= teams;
    p.per_cta = p.reduce ? teams / p.G * p.G : teams;
    const long long all = p.rows * p.G;                  // rows of groups
    // As many threads as an SM takes at most, and no more rows at a time than partial rows.  In the forward that is neither what a kernel's registers let in (two
    // to four CTAs of 256) nor a limit of its own, but the waves that it makes happen to suit the training size: without the cap 32768 rows of 32 groups of 64
    // take 76.6 instead of 73.8 us, of 5 groups of 128 28.9 instead of 32.8, of 20 groups of 80 65.6 instead of 68.4.
    // A backward keeps its parameters' sums, so its CTAs are no more than are resident (fp32, 16777 rows of 2 groups of 1000, with one too many:
    // 219 us, else 170).
    const int elements = q.vec * q.k;
    const int threads = forward ? 2048 : p.team > 32 ? 512 : 256 * bwd_ctas(elements, elements * (q.whole ? element : 4), p.gate != nullptr), ctas = threads > q.block ? threads / q.block : 1;
    const long long most_ctas = (long long)sm_count_of_current_device() * (ctas < 32 ? ctas : 32);
    long long grid = (all + p.per_cta - 1) / p.per_cta;
    if (!forward) {                        // four rows a team before there is a second CTA on an SM: each more is a partial row to add
        const long long four = (grid + 3) / 4, one = sm_count_of_current_device();
        grid = grid < one ? grid : four < one ? one : four;
    }
    grid = grid < most_ctas ? grid : most_ctas;
    if (p.reduce) {
        grid = grid < kMaxPartials ? grid : kMaxPartials;
        p.parallel = (int)(grid * (p.per_cta / p.G));
    } else {
        long long parallel = grid * p.per_cta / p.G;
        parallel = parallel > kMaxPartials ? kMaxPartials : parallel;
        parallel = parallel > p.rows ? p.rows : parallel < 1 ? 1 : parallel;
        p.parallel = (int)parallel;
        grid = (parallel * p.G + p.per_cta - 1) / p.per_cta;
    }
    q.grid = (int)grid;
    return q;
}
int aligned_to(std::initializer_list<const void*> ps, std::initializer_list<long long> strides, int element) {
    uintptr_t bits = 16;
    for (const void* q : ps) bits |= reinterpret_cast<uintptr_t>(q);
    for (long long s : strides) bits |= (uintptr_t)s * element;
    return (int)(bits & (0 - bits));
}
// Shared memory of a CTA: the rows to come of so many streams, and behind them the CTA's sums of the parameters' gradients.
template <typename T, int VEC, int K, bool kWhole, bool kAsync> constexpr size_t shared_bytes(int block, int streams, bool sums) {
    const size_t rows = Rows<T, VEC, K, kWhole, kAsync>::kBytes * streams * block, room = sums ? 2 * 256 * VEC * sizeof(float) : 0;
    return rows > room ? rows : room;
}
// `go` for the cut of a plan
template <typename T, typename Go> int dispatch(const Plan& q, const Problem& p, Go go) {
    constexpr int kWide = 16 / sizeof(T);
    typedef std::true_type Yes;
    typedef std::false_type No;
    typedef std::integral_constant<int, 0> Any;
    typedef std::integral_constant<int, kAnyTeam> Other;
    typedef std::integral_constant<int, 1> One;
    typedef std::integral_constant<int, 2> Two;
    typedef std::integral_constant<int, 4> Four;
    typedef std::integral_constant<int, 8> Eight;
    typedef std::integral_constant<int, 16> Sixteen;
    typedef std::integral_constant<int, 32> Warp;
    typedef std::integral_constant<int, kWide> Wide;
    const auto gated = [&](auto vec, auto k, auto whole, auto block, auto team) {
        return p.gate != nullptr ? go(vec, k, whole, block, team, Yes()) : go(vec, k, whole, block, team, No());
    };
    const bool block = p.team > 32, other = (p.team & (p.team - 1)) != 0;
    if (q.vec == kWide) {
        if (!block) {
            if (q.k == 2) return gated(Wide(), Two(), Yes(), No(), Warp());    // (more than 32 pieces)
            return p.team == 32   ? gated(Wide(), One(), Yes(), No(), Warp())
                   : p.team == 16 ? gated(Wide(), One(), Yes(), No(), Sixteen())
                   : p.team == 8  ? gated(Wide(), One(), Yes(), No(), Eight())
                   : other        ? gated(Wide(), One(), Yes(), No(), Other())
                                  : gated(Wide(), One(), Yes(), No(), Any());
        }
        if (q.k == 1) return gated(Wide(), One(), Yes(), Yes(), Any());
        if constexpr (sizeof(T) == 4) {                  // (in 16 bits two pieces a thread cover the widest group)
            if (q.k == 4) return gated(Wide(), Four(), Yes(), Yes(), Any());
        }
        return gated(Wide(), Two(), Yes(), Yes(), Any());
    }
    if (q.whole) {
        if (!block) return q.k == 8 ? gated(Two(), Eight(), Yes(), No(), Warp()) : other ? gated(Two(), Four(), Yes(), No(), Other()) : gated(Two(), Four(), Yes(), No(), Any());
        return q.k == 4 ? gated(Two(), Four(), Yes(), Yes(), Any()) : gated(Two(), Eight(), Yes(), Yes(), Any());
    }
    if (!block) return q.k == 8 ? gated(Two(), Eight(), No(), No(), Warp()) : other ? gated(Two(), Four(), No(), No(), Other()) : gated(Two(), Four(), No(), No(), Any());
    return q.k == 4 ? gated(Two(), Four(), No(), Yes(), Any()) : gated(Two(), Eight(), No(), Yes(), Any());
}
template <typename T> int fwd(cudaStream_t st, Problem p, void* y) {
    const Plan q = plan_of(p, sizeof(T), aligned_to({p.x, p.gate, y}, {p.x_stride, p.gate_stride, p.C}, sizeof(T)), true);
    return dispatch<T>(q, p, [&](auto vec, auto k, auto whole, auto block, auto team, auto gate) {
        const auto kern = group_norm_fwd_kernel<T, vec.value, k.value, whole.value, block.value, team.value, gate.value>;
        constexpr bool kAsync = vec.value == 8 && kAsyncRows<T, k.value, whole.value, block.value, true>;
        const size_t smem = shared_bytes<T, vec.value, k.value, whole.value, kAsync>(q.block, 1 + gate.value, false);       // (48 KB at most)
        kern<<<q.grid, q.block, smem, st>>>(p, (T*)y);
        return cudaGetLastError() == cudaSuccess ? B200WKV_OK : B200WKV_ELAUNCH;
    });
}
template <typename T>
int bwd(cudaStream_t st, Problem p, const void* gy, void* dx, void* dgate, void* dweight, void* dbias, float* partial) {
    const Plan q = plan_of(p, sizeof(T), aligned_to({p.x, p.gate, gy, dx, dgate}, {p.x_stride, p.gate_stride, p.C}, sizeof(T)), false);
    const bool params = dweight != nullptr || dbias != nullptr;
    if (!params) partial = nullptr;
    const int status = dispatch<T>(q, p, [&](auto vec, auto k, auto whole, auto block, auto team, auto gate) {
        const auto kern = group_norm_bwd_kernel<T, vec.value, k.value, whole.value, block.value, team.value, gate.value>;
        constexpr bool kAsync = vec.value == 8 && kAsyncRows<T, k.value, whole.value, block.value, false>;
        // (rows to come 36 KB at most, totals 16 to 64 KB for 256 threads, 64 KB for whole CTAs of 512)
        constexpr size_t kTotals = kTotalBytes<k.value * vec.value / 2, !(block.value && k.value * vec.value > 8)>;
        constexpr int kMost = block.value ? kMaxThreads : 256;
        static DeviceOnce once;
        if (!once.ok([&]() { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                         (int)(kTotals * kMost + shared_bytes<T, vec.value, k.value, whole.value, kAsync>(kMost, 2 + gate.value, !block.value))); }))
            return (int)B200WKV_ELAUNCH;
        const bool totals = partial != nullptr && p.rows > (long long)kChain * p.parallel;
        const size_t ring = shared_bytes<T, vec.value, k.value, whole.value, kAsync>(q.block, 2 + gate.value, p.reduce), smem = ring + (totals ? kTotals * q.block : 0);
        Problem pp = p;
        pp.totals = totals ? (int)ring : -1;
        kern<<<q.grid, q.block, smem, st>>>(pp, (const T*)gy, (T*)dx, (T*)dgate, partial);
        return cudaGetLastError() == cudaSuccess ? B200WKV_OK : B200WKV_ELAUNCH;
    });
    if (status != B200WKV_OK || !params) return status;
    const int n = p.reduce ? q.grid : p.parallel, f32 = p.weight.f32;
    return launch_behind(group_norm_sums_kernel, (2 * p.C + 31) / 32, 512, 0, st, (const float*)partial, n, p.C, f32, dweight, dbias) == cudaSuccess
               ? B200WKV_OK : B200WKV_ELAUNCH;
}
Problem problem(long long rows, int C, int groups, float eps, int act, const void* x, long long x_stride, const void* weight, const void* bias,
                int param_dtype, const void* gate, long long gate_stride) {
    const int f32 = param_dtype == B200WKV_F32;
    return {rows, C, groups, C / groups, act, eps, x, gate, x_stride, gate != nullptr ? gate_stride : 0, {weight, f32}, {bias, f32}, 0, 0, 0,
            aligned_to({weight, bias}, {}, 1) >= 16, -1, 0};
}
}  // namespace

size_t group_norm_workspace_bytes(long long rows, int C) { return (size_t)(rows < kMaxPartials ? rows : kMaxPartials) * 2 * C * sizeof(float); }

int group_norm_fwd(cudaStream_t st, int dtype, long long rows, int C, int groups, float eps, int act, const void* x, long long x_stride,
                   const void* weight, const void* bias, int param_dtype, const void* gate, long long gate_stride, void* y) {
    const Problem p = problem(rows, C, groups, eps, act, x, x_stride, weight, bias, param_dtype, gate, gate_stride);
    return dtype == B200WKV_F32 ? fwd<float>(st, p, y) : fwd<__nv_bfloat16>(st, p, y);
}
int group_norm_bwd(cudaStream_t st, int dtype, long long rows, int C, int groups, float eps, int act, const void* x, long long x_stride,
                   const void* weight, const void* bias, int param_dtype, const void* gate, long long gate_stride, const void* gy, void* dx,
                   void* dgate, void* dweight, void* dbias, void* workspace) {
    const Problem p = problem(rows, C, groups, eps, act, x, x_stride, weight, bias, param_dtype, gate, gate_stride);
    return dtype == B200WKV_F32 ? bwd<float>(st, p, gy, dx, dgate, dweight, dbias, (float*)workspace)
                                : bwd<__nv_bfloat16>(st, p, gy, dx, dgate, dweight, dbias, (float*)workspace);
}

}  // namespace b200wkv
