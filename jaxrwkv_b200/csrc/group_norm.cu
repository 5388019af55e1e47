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
    __device__ __forceinline__ float at(int c, float otherwise) const {
        return p == nullptr ? otherwise : f32 ? ((const float*)p)[c] : __bfloat162float(((const __nv_bfloat16*)p)[c]);
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
    int reduce;                            // teams of one group within a CTA are added up (per_cta is a multiple of G)
};

template <typename T, int VEC> __device__ __forceinline__ void load_piece(const T* p, float* v) {
    if constexpr (VEC == 1) {
        v[0] = to_f32(*p);
    } else if constexpr (sizeof(T) == 4) {
        const float4 q = *reinterpret_cast<const float4*>(p);
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
        const uint4 q = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}
template <typename T, int VEC> __device__ __forceinline__ void store_piece(T* p, const float* v) {
    if constexpr (VEC == 1) {
        *p = from_f32<T>(v[0]);
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
        uint4 q;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&q);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        *reinterpret_cast<uint4*>(p) = q;
    }
}

// act(z) and its derivative
template <typename T> __device__ __forceinline__ void activate(int act, float z, float& p, float& dp) {
    if (act == B200WKV_ACT_NONE) { p = z; dp = 1.f; return; }
    float s, r;
    sigmoid_pair<T>(z, s, r);
    p = act == B200WKV_ACT_SIGMOID ? s : z * s;
    dp = act == B200WKV_ACT_SIGMOID ? s * r : s * fmaf(z, r, 1.f);
}

// sums of two numbers over the team, the same in every thread of it
template <bool kBlock> __device__ __forceinline__ void team_sum(float& a, float& b, int team, float2* room) {
    const int width = kBlock ? 32 : team;
    for (int o = width / 2; o > 0; o /= 2) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (kBlock) {
        const int warps = blockDim.x / 32;
        __syncthreads();                   // the last sums have been read
        if (threadIdx.x % 32 == 0) room[threadIdx.x / 32] = make_float2(a, b);
        __syncthreads();
        a = 0.f; b = 0.f;
        for (int w = 0; w < warps; ++w) { a += room[w].x; b += room[w].y; }
    }
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

template <typename T, int VEC, int K, bool kBlock, bool kGate>
__global__ void __launch_bounds__(kBlock ? kMaxThreads : 256)
group_norm_fwd_kernel(const Problem p, T* __restrict__ y) {
    __shared__ float2 room[kBlock ? 32 : 1];
    const Place at(p);
    const int pieces = p.D / VEC, c0 = at.g * p.D;
    const float inv_d = 1.f / (float)p.D;
    float w[K][VEC], b[K][VEC];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const int d = (at.lane + k * p.team) * VEC + v;
            w[k][v] = d < p.D ? p.weight.at(c0 + d, 1.f) : 0.f;
            b[k][v] = d < p.D ? p.bias.at(c0 + d, 0.f) : 0.f;
        }
    // (teams without work go along: the sums take whole warps and CTAs)
    const long long steps = (p.rows + p.parallel - 1) / p.parallel;
    for (long long i = 0; i < steps; ++i) {
        const long long row = at.first + i * p.parallel;
        const bool on = at.at_work && row < p.rows;
        const T* const px = (const T*)p.x + row * p.x_stride + c0;
        const T* const pg = (const T*)p.gate + row * p.gate_stride + c0;
        float x[K][VEC], g[K][VEC], sum = 0.f, squares = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int piece = at.lane + k * p.team;
            if (on && piece < pieces) {
                load_piece<T, VEC>(px + piece * VEC, x[k]);
                if (kGate) load_piece<T, VEC>(pg + piece * VEC, g[k]);
            } else {
#pragma unroll
                for (int v = 0; v < VEC; ++v) x[k][v] = g[k][v] = 0.f;
            }
#pragma unroll
            for (int v = 0; v < VEC; ++v) sum += x[k][v];
        }
        team_sum<kBlock>(sum, squares, p.team, room);
        const float mean = sum * inv_d;
        squares = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                x[k][v] -= mean;
                if (at.lane + k * p.team < pieces) squares = fmaf(x[k][v], x[k][v], squares);
            }
        team_sum<kBlock>(squares, sum, p.team, room);
        const float rstd = 1.f / sqrtf(squares * inv_d + p.eps);
        T* const py = y + row * p.C + c0;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int piece = at.lane + k * p.team;
            if (!on || piece >= pieces) continue;
            float out[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float n = fmaf(x[k][v] * rstd, w[k][v], b[k][v]);
                float a, da;
                activate<T>(p.act, kGate ? g[k][v] : n, a, da);
                out[v] = kGate ? n * a : a;
            }
            store_piece<T, VEC>(py + piece * VEC, out);
        }
    }
}

template <typename T, int VEC, int K, bool kBlock, bool kGate>
__global__ void __launch_bounds__(kBlock ? kMaxThreads : 256)
group_norm_bwd_kernel(const Problem p, const T* __restrict__ gy, T* __restrict__ dx, T* __restrict__ dgate, float* __restrict__ partial) {
    __shared__ float2 room[kBlock ? 32 : 1];
    __shared__ float both[kBlock ? 1 : 256 * VEC];
    const Place at(p);
    const int pieces = p.D / VEC, c0 = at.g * p.D;
    const float inv_d = 1.f / (float)p.D;
    float w[K][VEC], b[K][VEC], dw[K][VEC], db[K][VEC];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const int d = (at.lane + k * p.team) * VEC + v;
            w[k][v] = d < p.D ? p.weight.at(c0 + d, 1.f) : 0.f;
            b[k][v] = d < p.D ? p.bias.at(c0 + d, 0.f) : 0.f;
            dw[k][v] = db[k][v] = 0.f;
        }
    const long long steps = (p.rows + p.parallel - 1) / p.parallel;
    for (long long i = 0; i < steps; ++i) {
        const long long row = at.first + i * p.parallel;
        const bool on = at.at_work && row < p.rows;
        const T* const px = (const T*)p.x + row * p.x_stride + c0;
        const T* const pg = (const T*)p.gate + row * p.gate_stride + c0;
        const size_t dense = (size_t)row * p.C + c0;
        float x[K][VEC], g[K][VEC], d[K][VEC], sum = 0.f, other = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int piece = at.lane + k * p.team;
            if (on && piece < pieces) {
                load_piece<T, VEC>(px + piece * VEC, x[k]);
                load_piece<T, VEC>(gy + dense + piece * VEC, d[k]);
                if (kGate) load_piece<T, VEC>(pg + piece * VEC, g[k]);
            } else {
#pragma unroll
                for (int v = 0; v < VEC; ++v) x[k][v] = g[k][v] = d[k][v] = 0.f;
            }
#pragma unroll
            for (int v = 0; v < VEC; ++v) sum += x[k][v];
        }
        team_sum<kBlock>(sum, other, p.team, room);
        const float mean = sum * inv_d;
        float squares = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                x[k][v] -= mean;
                if (at.lane + k * p.team < pieces) squares = fmaf(x[k][v], x[k][v], squares);
            }
        team_sum<kBlock>(squares, other, p.team, room);
        const float rstd = 1.f / sqrtf(squares * inv_d + p.eps);
        float s1 = 0.f, s2 = 0.f;          // of dxh and dxh xh
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int piece = at.lane + k * p.team;
            if (!on || piece >= pieces) continue;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float xh = x[k][v] * rstd, n = fmaf(xh, w[k][v], b[k][v]);
                float a, da;
                activate<T>(p.act, kGate ? g[k][v] : n, a, da);
                const float dn = d[k][v] * (kGate ? a : da);
                if (kGate) g[k][v] = d[k][v] * n * da;
                dw[k][v] = fmaf(dn, xh, dw[k][v]);
                db[k][v] += dn;
                const float dxh = dn * w[k][v];
                s1 += dxh;
                s2 = fmaf(dxh, xh, s2);
                x[k][v] = xh;
                d[k][v] = dxh;
            }
        }
        team_sum<kBlock>(s1, s2, p.team, room);
        s1 *= inv_d; s2 *= inv_d;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int piece = at.lane + k * p.team;
            if (!on || piece >= pieces) continue;
            if (kGate) store_piece<T, VEC>(dgate + dense + piece * VEC, g[k]);
#pragma unroll
            for (int v = 0; v < VEC; ++v) d[k][v] = rstd * (d[k][v] - s1 - x[k][v] * s2);
            store_piece<T, VEC>(dx + dense + piece * VEC, d[k]);
        }
    }
    if (partial == nullptr) return;
    // partial rows (parallel or one per CTA, 2, C): weight, bias
    if (!kBlock && p.reduce) {
        const int in_cta = threadIdx.x / p.team;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                __syncthreads();
#pragma unroll
                for (int v = 0; v < VEC; ++v) both[threadIdx.x * VEC + v] = which == 0 ? dw[k][v] : db[k][v];
                __syncthreads();
                if (in_cta < p.G && at.lane + k * p.team < pieces) {       // the first team of its group adds the others
                    for (int v = 0; v < VEC; ++v) {
                        float t = 0.f;
                        for (int j = in_cta; j < p.per_cta; j += p.G) t += both[(j * p.team + at.lane) * VEC + v];
                        partial[((size_t)blockIdx.x * 2 + which) * p.C + c0 + (at.lane + k * p.team) * VEC + v] = t;
                    }
                }
            }
        return;
    }
    if (!at.at_work) return;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int piece = at.lane + k * p.team;
        if (piece >= pieces) continue;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            partial[((size_t)at.first * 2) * p.C + c0 + piece * VEC + v] = dw[k][v];
            partial[((size_t)at.first * 2 + 1) * p.C + c0 + piece * VEC + v] = db[k][v];
        }
    }
}

// The partial rows' sums, in the parameters' type: a CTA owns 32 of the 2 C columns, its warps every sixteenth row, added in a fixed order.
__global__ void __launch_bounds__(512) group_norm_sums_kernel(const float* partial, int rows, int C, int f32, void* dweight, void* dbias) {
    __shared__ float part[16][32];
    wait_for_grid_in_front();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < 2 * C)
        for (int r = warp; r < rows; r += 64)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (r + 16 * j < rows) s[j] += partial[(size_t)(r + 16 * j) * 2 * C + c];
    part[warp][lane] = (s[0] + s[1]) + (s[2] + s[3]);
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
    const Plan q = plan_of(p, sizeof(T), on_16({p.x, p.gate, gy, dx, dgate}, {p.x_stride, p.gate_stride}, sizeof(T)), 4);
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
    return {rows, C, groups, C / groups, act, eps, x, gate, x_stride, gate != nullptr ? gate_stride : 0, {weight, f32}, {bias, f32}, 0, 0, 0, 0};
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
