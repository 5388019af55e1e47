// Group norm of rows of C channels, statistics per row and group of D = C / G consecutive channels, with an activation and,
// where a gate is given, a product with the activated gate (the output stage of RWKV-5, 5.2 and 6 has silu there):
//   xh = (x - mean) / sqrt(var + eps)   n = xh weight + bias   y = act(n), or n act(gate)
// Backward, dn = gy act'(n) or gy act(gate):
//   dgate = gy n act'(gate)   dxh = dn weight   dx = rstd (dxh - mean(dxh) - xh mean(dxh xh))
//   dweight = sum over rows of dn xh   dbias = sum over rows of dn
// The statistics are computed again in the backward (its x is read anyway), so nothing is kept.
//
// One pass over the rows, bound by memory.  A team of threads owns one group: a power of two of lanes of a warp with up to two
// 16-byte pieces of the row each, or a whole CTA where the group is wider than that.  The row's values stay in registers from
// the mean over the centred squares to the result.  A team keeps its group from row to row, so that weight and bias are read
// once and their gradients are added up in registers; they leave as partial rows, which a second kernel adds in a fixed order.
#include <initializer_list>
#include <type_traits>

#include "common.cuh"
#include "device_once.cuh"
#include "gate_math.cuh"
#include "host_calls.h"

namespace b200wkv {
namespace {

constexpr int kMaxPartials = 1024;         // partial rows of the parameters' gradients
constexpr int kMaxThreads = 1024;

struct Params {                            // weight or bias; p NULL: ones or zeros
    const void* p;
    int f32;
    // N from the c-th on, as pairs (N == 1: the same in both places); 16-byte loads where `vectors`
    template <int N> __device__ __forceinline__ void load(int c, bool vectors, float otherwise, F2* to) const {
        if (p == nullptr) {
#pragma unroll
            for (int i = 0; i < (N + 1) / 2; ++i) to[i] = both(otherwise);
        } else if constexpr (N == 1) {
            to[0] = both(f32 ? ((const float*)p)[c] : __bfloat162float(((const __nv_bfloat16*)p)[c]));
        } else if (f32 && vectors) {
#pragma unroll
            for (int i = 0; i < N / 4; ++i) {
                const float4 q = ((const float4*)((const float*)p + c))[i];
                to[2 * i] = make_f2(q.x, q.y);
                to[2 * i + 1] = make_f2(q.z, q.w);
            }
        } else if (vectors) {
#pragma unroll
            for (int i = 0; i < N / 4; ++i) {
                const uint2 q = ((const uint2*)((const __nv_bfloat16*)p + c))[i];
                to[2 * i] = unpack_pair(q.x);
                to[2 * i + 1] = unpack_pair(q.y);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N / 2; ++i)
                to[i] = f32 ? make_f2(((const float*)p)[c + 2 * i], ((const float*)p)[c + 2 * i + 1])
                            : make_f2(__bfloat162float(((const __nv_bfloat16*)p)[c + 2 * i]), __bfloat162float(((const __nv_bfloat16*)p)[c + 2 * i + 1]));
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
    int reduce;                            // teams of one group within a CTA are added up (per_cta is a multiple of G)
};

// A piece of a row as it lies in memory: VEC elements, 16 bytes, or one.  As pairs of floats a single element stands in both places.
template <typename T, int VEC> struct Piece { uint4 q; };
template <typename T> struct Piece<T, 1> { T q; };
template <typename T, int VEC> __device__ __forceinline__ void unpack(const Piece<T, VEC>& r, F2* v) {
    if constexpr (VEC == 1) v[0] = both(to_f32(r.q));
    else if constexpr (sizeof(T) == 4) {
        v[0] = make_f2(__uint_as_float(r.q.x), __uint_as_float(r.q.y));
        v[1] = make_f2(__uint_as_float(r.q.z), __uint_as_float(r.q.w));
    } else {
        v[0] = unpack_pair(r.q.x); v[1] = unpack_pair(r.q.y); v[2] = unpack_pair(r.q.z); v[3] = unpack_pair(r.q.w);
    }
}
template <typename T, int VEC> __device__ __forceinline__ void store_piece(T* p, const F2* v) {
    if constexpr (VEC == 1) {
        *p = from_f32<T>(parts(v[0]).x);
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<ulonglong2*>(p) = make_ulonglong2(v[0].v, v[1].v);
    } else {
        uint4 q;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&q);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 t = parts(v[i]);
            h[i] = __floats2bfloat162_rn(t.x, t.y);
        }
        *reinterpret_cast<uint4*>(p) = q;
    }
}
template <int VEC> __device__ __forceinline__ float sum_of(F2 v) {
    const float2 t = parts(v);
    return VEC == 1 ? t.x : t.x + t.y;
}

// act(z), and its derivative where it is asked for
template <typename T, int kAct> __device__ __forceinline__ void activate(F2 z, F2& p, F2& dp) {
    if (kAct == B200WKV_ACT_NONE) { p = z; dp = both(1.f); return; }
    F2 s, r;
    sigmoid_pair<T>(z, s, r);
    p = kAct == B200WKV_ACT_SIGMOID ? s : mul2(z, s);
    dp = kAct == B200WKV_ACT_SIGMOID ? mul2(s, r) : mul2(s, fma2(z, r, both(1.f)));
}

// sum over the team, the same in every thread of it
template <bool kBlock> __device__ __forceinline__ float team_sum(float a, int team, float* room) {
#pragma unroll
    for (int o = 16; o > 0; o /= 2)
        if (kBlock || team > o) a += __shfl_xor_sync(0xffffffffu, a, o);
    if (kBlock) {
        const int warps = blockDim.x / 32;
        __syncthreads();                   // the last sums have been read
        if (threadIdx.x % 32 == 0) room[threadIdx.x / 32] = a;
        __syncthreads();
        a = 0.f;
        for (int w = 0; w < warps; ++w) a += room[w];
    }
    return a;
}

// Where a thread's team works: group g, rows first, first + parallel, ...; none of them where `at_work` is false
struct Place {
    int g, lane;
    long long first;
    bool at_work;
    __device__ __forceinline__ Place(const Problem& p) {
        const int in_cta = threadIdx.x / p.team, q = blockIdx.x * p.per_cta + in_cta;
        lane = threadIdx.x % p.team;
        g = q % p.G;
        first = q / p.G;
        at_work = in_cta < p.per_cta && first < p.parallel;
    }
};

// Registers: weight, bias and a row's values; 4 CTAs an SM where the team is a part of a warp
template <typename T, int VEC, int K, bool kBlock, bool kGate>
__global__ void __launch_bounds__(kBlock ? kMaxThreads : 256, kBlock ? 1 : VEC * K > 8 || VEC == 1 && K == 8 ? 2 : 4)
group_norm_fwd_kernel(const Problem p, T* __restrict__ y) {
    constexpr int kPairs = (VEC + 1) / 2;
    __shared__ float room[kBlock ? 32 : 1];
    const Place at(p);
    const int pieces = p.D / VEC, c = at.g * p.D + at.lane * VEC, step = p.team * VEC;      // channels from piece to piece
    const float inv_d = 1.f / (float)p.D;
    F2 w[K][kPairs], b[K][kPairs];
    Piece<T, VEC> rx[K] = {}, rg[K] = {};
    bool there[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        there[k] = at.at_work && at.lane + k * p.team < pieces;
        if (there[k]) {
            p.weight.load<VEC>(c + k * step, p.param_vectors, 1.f, w[k]);
            p.bias.load<VEC>(c + k * step, p.param_vectors, 0.f, b[k]);
        } else {
#pragma unroll
            for (int i = 0; i < kPairs; ++i) w[k][i] = b[k][i] = both(0.f);
        }
    }
    const T* px = (const T*)p.x + at.first * p.x_stride + c;
    const T* pg = kGate ? (const T*)p.gate + at.first * p.gate_stride + c : nullptr;
    T* py = y + at.first * p.C + c;
    const auto read = [&](long long row) {
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (there[k] && row < p.rows) {
                rx[k] = *(const Piece<T, VEC>*)(px + k * step);
                if (kGate) rg[k] = *(const Piece<T, VEC>*)(pg + k * step);
            }
        px += p.parallel * p.x_stride;
        if (kGate) pg += p.parallel * p.gate_stride;
    };
    read(at.first);
    // (teams without work go along: the sums take whole warps and CTAs)
    const long long steps = (p.rows + p.parallel - 1) / p.parallel;
    long long row = at.first;
    for (long long i = 0; i < steps; ++i, row += p.parallel, py += (long long)p.parallel * p.C) {
        F2 x[K][kPairs], g[K][kPairs], sums = both(0.f);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            unpack<T, VEC>(rx[k], x[k]);
            if (kGate) unpack<T, VEC>(rg[k], g[k]);
#pragma unroll
            for (int j = 0; j < kPairs; ++j) sums = add2(sums, x[k][j]);
        }
        read(row + p.parallel);
        const float mean = team_sum<kBlock>(sum_of<VEC>(sums), p.team, room) * inv_d;
        sums = both(0.f);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            F2 squares = both(0.f);
#pragma unroll
            for (int j = 0; j < kPairs; ++j) {
                x[k][j] = add2(x[k][j], both(-mean));
                squares = fma2(x[k][j], x[k][j], squares);
            }
            if (there[k]) sums = add2(sums, squares);
        }
        const float rstd = rsqrtf(team_sum<kBlock>(sum_of<VEC>(sums), p.team, room) * inv_d + p.eps);
        const auto finish = [&](auto act) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (!there[k] || row >= p.rows) continue;
                F2 out[kPairs];
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    const F2 n = fma2(mul2(x[k][j], both(rstd)), w[k][j], b[k][j]);
                    F2 a, da;
                    activate<T, act.value>(kGate ? g[k][j] : n, a, da);
                    out[j] = kGate ? mul2(n, a) : a;
                }
                store_piece<T, VEC>(py + k * step, out);
            }
        };
        if (p.act == B200WKV_ACT_SILU) finish(std::integral_constant<int, B200WKV_ACT_SILU>());
        else if (p.act == B200WKV_ACT_SIGMOID) finish(std::integral_constant<int, B200WKV_ACT_SIGMOID>());
        else finish(std::integral_constant<int, B200WKV_ACT_NONE>());
    }
}

template <typename T, int VEC, int K, bool kBlock, bool kGate>
__global__ void __launch_bounds__(kBlock ? kMaxThreads : 256, kBlock ? 1 : VEC * K > 8 || VEC == 1 && K == 8 ? 1 : 2)
group_norm_bwd_kernel(const Problem p, const T* __restrict__ gy, T* __restrict__ dx, T* __restrict__ dgate, float* __restrict__ partial) {
    constexpr int kPairs = (VEC + 1) / 2;
    __shared__ float room[kBlock ? 32 : 1];
    __shared__ float both_sums[kBlock ? 1 : 256 * VEC];
    const Place at(p);
    const int pieces = p.D / VEC, c = at.g * p.D + at.lane * VEC, step = p.team * VEC;
    const float inv_d = 1.f / (float)p.D;
    F2 w[K][kPairs], b[K][kPairs], dw[K][kPairs], db[K][kPairs];
    Piece<T, VEC> rx[K] = {}, rg[K] = {}, rd[K] = {};
    bool there[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        there[k] = at.at_work && at.lane + k * p.team < pieces;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) w[k][i] = b[k][i] = dw[k][i] = db[k][i] = both(0.f);
        if (there[k]) {
            p.weight.load<VEC>(c + k * step, p.param_vectors, 1.f, w[k]);
            p.bias.load<VEC>(c + k * step, p.param_vectors, 0.f, b[k]);
        }
    }
    const T* px = (const T*)p.x + at.first * p.x_stride + c;
    const T* pg = kGate ? (const T*)p.gate + at.first * p.gate_stride + c : nullptr;
    const T* pd = gy + at.first * p.C + c;
    long long dense = at.first * p.C + c;
    const auto read = [&](long long row) {
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (there[k] && row < p.rows) {
                rx[k] = *(const Piece<T, VEC>*)(px + k * step);
                rd[k] = *(const Piece<T, VEC>*)(pd + k * step);
                if (kGate) rg[k] = *(const Piece<T, VEC>*)(pg + k * step);
            }
        px += p.parallel * p.x_stride;
        pd += (long long)p.parallel * p.C;
        if (kGate) pg += p.parallel * p.gate_stride;
    };
    read(at.first);
    const long long steps = (p.rows + p.parallel - 1) / p.parallel;
    long long row = at.first;
    for (long long i = 0; i < steps; ++i, row += p.parallel, dense += (long long)p.parallel * p.C) {
        const bool on = row < p.rows;
        F2 x[K][kPairs], g[K][kPairs], d[K][kPairs], sums = both(0.f);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            unpack<T, VEC>(rx[k], x[k]);
            unpack<T, VEC>(rd[k], d[k]);
            if (kGate) unpack<T, VEC>(rg[k], g[k]);
#pragma unroll
            for (int j = 0; j < kPairs; ++j) sums = add2(sums, x[k][j]);
        }
        read(row + p.parallel);
        const float mean = team_sum<kBlock>(sum_of<VEC>(sums), p.team, room) * inv_d;
        sums = both(0.f);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            F2 squares = both(0.f);
#pragma unroll
            for (int j = 0; j < kPairs; ++j) {
                x[k][j] = add2(x[k][j], both(-mean));
                squares = fma2(x[k][j], x[k][j], squares);
            }
            if (there[k]) sums = add2(sums, squares);
        }
        const float rstd = rsqrtf(team_sum<kBlock>(sum_of<VEC>(sums), p.team, room) * inv_d + p.eps);
        F2 s1 = both(0.f), s2 = both(0.f);          // of dxh and dxh xh
        const auto gradients = [&](auto act) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (!there[k] || !on) continue;
#pragma unroll
                for (int j = 0; j < kPairs; ++j) {
                    const F2 xh = mul2(x[k][j], both(rstd)), n = fma2(xh, w[k][j], b[k][j]);
                    F2 a, da;
                    activate<T, act.value>(kGate ? g[k][j] : n, a, da);
                    const F2 dn = mul2(d[k][j], kGate ? a : da);
                    if (kGate) g[k][j] = mul2(mul2(d[k][j], n), da);
                    dw[k][j] = fma2(dn, xh, dw[k][j]);
                    db[k][j] = add2(db[k][j], dn);
                    const F2 dxh = mul2(dn, w[k][j]);
                    s1 = add2(s1, dxh);
                    s2 = fma2(dxh, xh, s2);
                    x[k][j] = xh;
                    d[k][j] = dxh;
                }
            }
        };
        if (p.act == B200WKV_ACT_SILU) gradients(std::integral_constant<int, B200WKV_ACT_SILU>());
        else if (p.act == B200WKV_ACT_SIGMOID) gradients(std::integral_constant<int, B200WKV_ACT_SIGMOID>());
        else gradients(std::integral_constant<int, B200WKV_ACT_NONE>());
        const float m1 = team_sum<kBlock>(sum_of<VEC>(s1), p.team, room) * inv_d, m2 = team_sum<kBlock>(sum_of<VEC>(s2), p.team, room) * inv_d;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (!there[k] || !on) continue;
            if (kGate) store_piece<T, VEC>(dgate + dense + k * step, g[k]);
#pragma unroll
            for (int j = 0; j < kPairs; ++j) d[k][j] = mul2(fma2(x[k][j], both(-m2), add2(d[k][j], both(-m1))), both(rstd));
            store_piece<T, VEC>(dx + dense + k * step, d[k]);
        }
    }
    if (partial == nullptr) return;
    // partial rows (parallel or one per CTA, 2, C): weight, bias
    const auto of = [](const F2* v, int i) { return i % 2 == 0 ? parts(v[i / 2]).x : parts(v[i / 2]).y; };
    if (!kBlock && p.reduce) {
        const int in_cta = threadIdx.x / p.team;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                __syncthreads();
#pragma unroll
                for (int v = 0; v < VEC; ++v) both_sums[threadIdx.x * VEC + v] = of(which == 0 ? dw[k] : db[k], v);
                __syncthreads();
                if (in_cta < p.G && there[k])              // the first team of its group adds the others
                    for (int v = 0; v < VEC; ++v) {
                        float t = 0.f;
                        for (int j = in_cta; j < p.per_cta; j += p.G) t += both_sums[(j * p.team + at.lane) * VEC + v];
                        partial[((size_t)blockIdx.x * 2 + which) * p.C + c + k * step + v] = t;
                    }
            }
        return;
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (there[k]) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                partial[((size_t)at.first * 2) * p.C + c + k * step + v] = of(dw[k], v);
                partial[((size_t)at.first * 2 + 1) * p.C + c + k * step + v] = of(db[k], v);
            }
        }
}

// The partial rows' sums, in the parameters' type: a CTA owns 32 of the 2 C columns, its warps every sixteenth row, added in a fixed order.
__global__ void __launch_bounds__(512) group_norm_sums_kernel(const float* partial, int rows, int C, int f32, void* dweight, void* dbias) {
    __shared__ float part[16][32];
    wait_for_grid_in_front();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float s[8] = {};
    if (c < 2 * C)
        for (int r = warp; r < rows; r += 128)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (r + 16 * j < rows) s[j] += partial[(size_t)(r + 16 * j) * 2 * C + c];
    part[warp][lane] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    __syncthreads();
    if (warp != 0 || c >= 2 * C) return;
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) t += part[w][lane];
    void* const to = c < C ? dweight : dbias;
    if (to == nullptr) return;
    const int at = c < C ? c : c - C;
    if (f32) ((float*)to)[at] = t;
    else ((__nv_bfloat16*)to)[at] = __float2bfloat16_rn(t);
}

// How a call is cut: pieces of 16 bytes where rows and group fit them, else single elements; a team as narrow as covers the group.
struct Plan {
    int vec, k, block, grid;
};
Plan plan_of(Problem& p, int element, bool aligned, int ctas_per_sm) {
    Plan q;
    const int wide = 16 / element;
    q.vec = aligned && p.D % wide == 0 && p.C % wide == 0 ? wide : 1;
    const int pieces = p.D / q.vec, most = q.vec == 1 ? 8 : 2;
    if (pieces <= 32 * most) {
        q.k = pieces <= 32 ? 1 : q.vec == 1 ? (pieces <= 64 ? 2 : 8) : 2;
        p.team = 1;
        while (p.team * q.k < pieces) p.team *= 2;
        q.block = 256;
    } else {
        q.k = pieces <= kMaxThreads ? 1 : q.vec == 1 ? 8 : 2;
        q.block = ((pieces + q.k - 1) / q.k + 31) / 32 * 32;
        p.team = q.block;
    }
    const int teams = q.block / p.team;
    p.reduce = p.G * 4 <= teams;
    p.per_cta = p.reduce ? teams / p.G * p.G : teams;
    const long long all = p.rows * p.G;                  // rows of groups
    const long long most_ctas = (long long)sm_count_of_current_device() * ctas_per_sm;
    long long grid = (all + p.per_cta - 1) / p.per_cta;
    grid = grid < most_ctas ? grid : most_ctas;
    if (p.reduce) {
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
bool on_16(std::initializer_list<const void*> ps, std::initializer_list<long long> strides, int element) {
    uintptr_t bits = 0;
    for (const void* q : ps) bits |= reinterpret_cast<uintptr_t>(q);
    for (long long s : strides) bits |= (uintptr_t)s * element;
    return bits % 16 == 0;
}
// `go` for the cut of a plan
template <typename T, typename Go> int dispatch(const Plan& q, const Problem& p, Go go) {
    constexpr int kWide = 16 / sizeof(T);
    typedef std::integral_constant<int, 1> One;
    typedef std::integral_constant<int, 2> Two;
    typedef std::integral_constant<int, 8> Eight;
    typedef std::integral_constant<int, kWide> Wide;
    const auto gated = [&](auto vec, auto k, auto block) {
        return p.gate != nullptr ? go(vec, k, block, std::true_type()) : go(vec, k, block, std::false_type());
    };
    const auto shaped = [&](auto vec, auto k) {
        return p.team > 32 ? gated(vec, k, std::true_type()) : gated(vec, k, std::false_type());
    };
    if (q.vec > 1) return q.k == 1 ? shaped(Wide(), One()) : shaped(Wide(), Two());
    return q.k == 1 ? shaped(One(), One()) : q.k == 2 ? gated(One(), Two(), std::false_type()) : shaped(One(), Eight());
}
template <typename T> int fwd(cudaStream_t st, Problem p, void* y) {
    const Plan q = plan_of(p, sizeof(T), on_16({p.x, p.gate, y}, {p.x_stride, p.gate_stride}, sizeof(T)), 8);
    return dispatch<T>(q, p, [&](auto vec, auto k, auto block, auto gate) {
        group_norm_fwd_kernel<T, vec.value, k.value, block.value, gate.value><<<q.grid, q.block, 0, st>>>(p, (T*)y);
        return cudaGetLastError() == cudaSuccess ? B200WKV_OK : B200WKV_ELAUNCH;
    });
}
template <typename T>
int bwd(cudaStream_t st, Problem p, const void* gy, void* dx, void* dgate, void* dweight, void* dbias, float* partial) {
    const Plan q = plan_of(p, sizeof(T), on_16({p.x, p.gate, gy, dx, dgate}, {p.x_stride, p.gate_stride}, sizeof(T)), 2);
    const bool params = dweight != nullptr || dbias != nullptr;
    if (!params) partial = nullptr;
    const int status = dispatch<T>(q, p, [&](auto vec, auto k, auto block, auto gate) {
        group_norm_bwd_kernel<T, vec.value, k.value, block.value, gate.value><<<q.grid, q.block, 0, st>>>(p, (const T*)gy, (T*)dx, (T*)dgate, partial);
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
            on_16({weight, bias}, {}, 4), 0};
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
