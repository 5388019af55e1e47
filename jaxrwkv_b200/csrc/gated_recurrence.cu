// Gated linear recurrence, one number of state per channel, fp32 arithmetic and state:
//   gate "sigmoid":  a = sigmoid(f)      u = (1 - a) x
//   gate "decay":    a = exp(-exp(f))    u = x             (f: the raw log-log decay, as RWKV-7's w)
//   h_t = (start_t ? 0 : a_t h_{t-1}) + u_t     out_t = h_t     s_out = h_{length-1}
// Both gates lie in [0, 1], so a product of them over any stretch of tokens cannot overflow.
//
// The recurrence is associative: a stretch of tokens acts on the state entering it as h -> A h + b.  A CTA of eight warps owns
// 32 V channels of one sequence, each warp consecutive segments of kSeg tokens, and the CTAs of a cluster own consecutive tiles:
//   1. every warp reduces its segment to (A, b), its gates staying in registers;
//   2. these are combined in order, inside the CTA through shared memory and then across the cluster through distributed
//      shared memory, which gives every segment the state entering it;
//   3. every warp walks its segment from that state and writes the outputs.
// The cluster then moves on by its tiles with the combined state as carry.
//
// Backward: dh_t = gy_t + [t == length-1] gs + c_{t+1},  c_t = start_t ? 0 : a_t dh_t.  The states are recomputed from the
// state entering each tile, which the forward keeps (4 bytes per tile and channel); c runs over the segments from the last to
// the first with the same products A.
//
// A start flag cuts by a select, not by a factor of 0: what is no number in front of it ends there.
#include <cooperative_groups.h>

#include <initializer_list>

#include "common.cuh"
#include "device_once.cuh"
#include "gate_math.cuh"
#include "host_calls.h"

namespace b200wkv {
namespace {
namespace cg = cooperative_groups;

constexpr int kSeg = 8;                    // tokens of a warp's segment
constexpr int kWarps = 8;
constexpr int kTile = kSeg * kWarps;       // tokens of a CTA's tile: a checkpoint each
constexpr int kMaxCluster = 8;

// V channels, as they lie in memory
template <typename T, int V> struct Raw;
template <> struct Raw<float, 1> { float q; };
template <> struct Raw<float, 2> { float2 q; };
template <> struct Raw<__nv_bfloat16, 1> { __nv_bfloat16 q; };
template <> struct Raw<__nv_bfloat16, 2> { uint32_t q; };
__device__ __forceinline__ float channel(const Raw<float, 1>& r, int) { return r.q; }
__device__ __forceinline__ float channel(const Raw<float, 2>& r, int v) { return v == 0 ? r.q.x : r.q.y; }
__device__ __forceinline__ float channel(const Raw<__nv_bfloat16, 1>& r, int) { return __bfloat162float(r.q); }
__device__ __forceinline__ float channel(const Raw<__nv_bfloat16, 2>& r, int v) { return __uint_as_float(v == 0 ? r.q << 16 : r.q & 0xffff0000u); }
template <typename T, int V> __device__ __forceinline__ Raw<T, V> load_raw(const T* p) { return *reinterpret_cast<const Raw<T, V>*>(p); }
template <int V> __device__ __forceinline__ void store_out(float* p, const float* h) {
    if constexpr (V == 2) *reinterpret_cast<float2*>(p) = make_float2(h[0], h[1]);
    else *p = h[0];
}
template <int V> __device__ __forceinline__ void store_out(__nv_bfloat16* p, const float* h) {
    if constexpr (V == 2) *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(h[0], h[1]);
    else *p = __float2bfloat16_rn(h[0]);
}

constexpr int kSigmoidGate = B200WKV_GATE_SIGMOID;
// The gate a, and what the backward needs of it: `w`, for the sigmoid 1 - a (to full relative precision), for the decay -da/df.
template <typename T, int kGate> __device__ __forceinline__ void gate_of(float f, float& a, float& w) {
    if (kGate == kSigmoidGate) {
        sigmoid_pair<T>(f, a, w);
    } else {
        // (accurate in 16 bits too: the state sums 1 / (1 - a) tokens, and an error of a is that much larger in it)
        const float e = expf(f);
        a = expf(-e);
        w = a == 0.f ? 0.f : e * a;        // (e may be infinite then)
    }
}

// start flags of the segment that begins at t0 as a bit mask (bit i = token t0 + i)
__device__ __forceinline__ uint32_t segment_flags(const uint8_t* ns, int t0, int Tlen, int lane) {
    const bool f = ns != nullptr && lane < kSeg && t0 + lane < Tlen && ns[t0 + lane] != 0;
    return __ballot_sync(0xffffffffu, f);
}

struct Stream {                            // rows of C adjacent channels
    const void* p;
    long long batch, token;                // strides in elements
};
struct Problem {
    int T, C, slabs;
    Stream x, f;
    const float* s0;
    const uint32_t* length;
    const uint8_t* starts;
};

// (A, b) of the segments and of the CTA; `cut`: a start flag lies inside
template <int V> struct Summaries {
    float A[kWarps][32 * V], b[kWarps][32 * V];
    float cta_A[32 * V], cta_b[32 * V];
    int cut[kWarps], cta_cut;
};

template <typename T, int V, int kGate>
__global__ void __launch_bounds__(kWarps * 32, 2)
gated_fwd_kernel(const Problem p, T* __restrict__ y, float* __restrict__ s_out, float* __restrict__ ckpt) {
    __shared__ Summaries<V> sm;
    const cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int unit = blockIdx.x / ranks, bi = unit / p.slabs, c = ((unit % p.slabs) * 32 + lane) * V;
    const bool live = c < p.C;
    const int cc = live ? c : 0;
    const int L = p.length != nullptr ? (int)min(p.length[bi], (uint32_t)p.T) : p.T;
    const int tiles = (p.T + kTile - 1) / kTile;
    const size_t so = (size_t)bi * p.C + cc;
    float carry[V];                        // state entering the tiles at hand
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = p.s0 != nullptr ? p.s0[so + v] : 0.f;
    if (L == 0 && warp == 0 && rank == 0 && live) {
#pragma unroll
        for (int v = 0; v < V; ++v) s_out[so + v] = carry[v];
    }
    const T* const px = (const T*)p.x.p + bi * p.x.batch + cc;
    const T* const pf = (const T*)p.f.p + bi * p.f.batch + cc;
    T* const py = y + (size_t)bi * p.T * p.C + cc;
    const uint8_t* const ns = p.starts != nullptr ? p.starts + (size_t)bi * p.T : nullptr;
    for (int tile0 = 0; tile0 < tiles; tile0 += ranks) {
        const int tile = tile0 + rank, t0 = tile * kTile + warp * kSeg, n = max(0, min(kSeg, p.T - t0));
        // 1. summary; tokens behind the end leave the state as it is
        float a[kSeg][V], u[kSeg][V], A[V], b[V];
        if (n > 0) {
            Raw<T, V> rx[kSeg], rf[kSeg];
#pragma unroll
            for (int i = 0; i < kSeg; ++i) {
                const size_t t = (size_t)(t0 + min(i, n - 1));
                rx[i] = load_raw<T, V>(px + t * p.x.token);
                rf[i] = load_raw<T, V>(pf + t * p.f.token);
            }
#pragma unroll
            for (int i = 0; i < kSeg; ++i)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    float w;
                    gate_of<T, kGate>(channel(rf[i], v), a[i][v], w);
                    u[i][v] = kGate == kSigmoidGate ? w * channel(rx[i], v) : channel(rx[i], v);
                }
        }
        const uint32_t starts = segment_flags(ns, t0, p.T, lane);
#pragma unroll
        for (int v = 0; v < V; ++v) { A[v] = 1.f; b[v] = 0.f; }
#pragma unroll
        for (int i = 0; i < kSeg; ++i)
            if (i < n) {
                const bool start = (starts >> i) & 1u;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    b[v] = start ? u[i][v] : fmaf(a[i][v], b[v], u[i][v]);
                    A[v] = start ? 0.f : A[v] * a[i][v];
                }
            }
#pragma unroll
        for (int v = 0; v < V; ++v) { sm.A[warp][lane * V + v] = A[v]; sm.b[warp][lane * V + v] = b[v]; }
        if (lane == 0) sm.cut[warp] = starts != 0;
        __syncthreads();
        // 2. what the segments in front of this one make of the state entering the tile, and what the whole tile does
        float qA[V], qb[V];
        bool cut = false, own_cut = false;
#pragma unroll
        for (int v = 0; v < V; ++v) { qA[v] = 1.f; qb[v] = 0.f; }
#pragma unroll
        for (int j = 0; j < kWarps; ++j) {
            if (j == warp) {
                own_cut = cut;
#pragma unroll
                for (int v = 0; v < V; ++v) { A[v] = qA[v]; b[v] = qb[v]; }
            }
            const bool cj = sm.cut[j] != 0;
            cut |= cj;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float Aj = sm.A[j][lane * V + v], bj = sm.b[j][lane * V + v];
                qb[v] = cj ? bj : fmaf(Aj, qb[v], bj);
                qA[v] = cj ? 0.f : Aj * qA[v];
            }
        }
        if (ranks > 1) {
            if (warp == 0) {
#pragma unroll
                for (int v = 0; v < V; ++v) { sm.cta_A[lane * V + v] = qA[v]; sm.cta_b[lane * V + v] = qb[v]; }
                if (lane == 0) sm.cta_cut = cut;
            }
            cluster.sync();
        }
        float h[V];
        for (int q = 0; q < ranks; ++q) {
            const bool own = q == rank;
            const Summaries<V>* from = own ? &sm : cluster.map_shared_rank(&sm, q);
            const bool cq = own ? cut : from->cta_cut != 0;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float Aq = own ? qA[v] : from->cta_A[lane * V + v], bq = own ? qb[v] : from->cta_b[lane * V + v];
                if (own) h[v] = carry[v];
                carry[v] = cq ? bq : fmaf(Aq, carry[v], bq);
            }
        }
        if (ckpt != nullptr && warp == 0 && n > 0 && live) store_out<V>(ckpt + ((size_t)bi * tiles + tile) * p.C + cc, h);
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = own_cut ? b[v] : fmaf(A[v], h[v], b[v]);
        // 3. outputs
#pragma unroll
        for (int i = 0; i < kSeg; ++i)
            if (i < n) {
                const bool start = (starts >> i) & 1u;
#pragma unroll
                for (int v = 0; v < V; ++v) h[v] = start ? u[i][v] : fmaf(a[i][v], h[v], u[i][v]);
                if (live) {
                    store_out<V>(py + (size_t)(t0 + i) * p.C, h);
                    if (t0 + i == L - 1) store_out<V>(s_out + so, h);
                }
            }
        if (ranks > 1) cluster.sync(); else __syncthreads();   // the summaries are read before the next ones are written
    }
}

template <typename T, int V, int kGate>
__global__ void __launch_bounds__(kWarps * 32, 2)
gated_bwd_kernel(const Problem p, const T* __restrict__ gy, const float* __restrict__ gs, const float* __restrict__ ckpt,
                 T* __restrict__ dx, T* __restrict__ df, float* __restrict__ ds0) {
    __shared__ Summaries<V> sm;
    __shared__ float back[kWarps][32 * V];     // what a segment sends to the one in front of it when nothing comes from behind
    const cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int unit = blockIdx.x / ranks, bi = unit / p.slabs, c = ((unit % p.slabs) * 32 + lane) * V;
    const bool live = c < p.C;
    const int cc = live ? c : 0;
    const int L = p.length != nullptr ? (int)min(p.length[bi], (uint32_t)p.T) : p.T;
    const int tiles = (p.T + kTile - 1) / kTile;
    const size_t so = (size_t)bi * p.C + cc, base = (size_t)bi * p.T * p.C + cc;
    float carry[V], gstate[V];             // c entering the tiles at hand from behind; the returned state's cotangent
#pragma unroll
    for (int v = 0; v < V; ++v) { carry[v] = 0.f; gstate[v] = gs != nullptr ? gs[so + v] : 0.f; }
    const T* const px = (const T*)p.x.p + bi * p.x.batch + cc;
    const T* const pf = (const T*)p.f.p + bi * p.f.batch + cc;
    const uint8_t* const ns = p.starts != nullptr ? p.starts + (size_t)bi * p.T : nullptr;
    for (int tile0 = (tiles - 1) / ranks * ranks; tile0 >= 0; tile0 -= ranks) {
        const int tile = tile0 + rank, t0 = tile * kTile + warp * kSeg, n = max(0, min(kSeg, p.T - t0));
        float a[kSeg][V], w[kSeg][V], x[kSeg][V], g[kSeg][V], A[V], b[V], h[V];
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = 0.f;
        if (n > 0) {
            Raw<T, V> rx[kSeg], rf[kSeg], rg[kSeg];
#pragma unroll
            for (int i = 0; i < kSeg; ++i) {
                const size_t t = (size_t)(t0 + min(i, n - 1));
                rx[i] = load_raw<T, V>(px + t * p.x.token);
                rf[i] = load_raw<T, V>(pf + t * p.f.token);
                if (gy != nullptr) rg[i] = load_raw<T, V>(gy + base + t * p.C);
            }
            const float* const q = ckpt + ((size_t)bi * tiles + tile) * p.C + cc;
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = q[v];
#pragma unroll
            for (int i = 0; i < kSeg; ++i)
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    gate_of<T, kGate>(channel(rf[i], v), a[i][v], w[i][v]);
                    x[i][v] = channel(rx[i], v);
                    g[i][v] = gy != nullptr ? channel(rg[i], v) : 0.f;
                    if (t0 + i == L - 1) g[i][v] += gstate[v];
                }
        }
        const uint32_t starts = segment_flags(ns, t0, p.T, lane);
        // 1. the segment's summary for the states, and what it sends to the front
        float send[V];
#pragma unroll
        for (int v = 0; v < V; ++v) { A[v] = 1.f; b[v] = 0.f; send[v] = 0.f; }
#pragma unroll
        for (int i = 0; i < kSeg; ++i)
            if (i < n) {
                const bool start = (starts >> i) & 1u;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float u = kGate == kSigmoidGate ? w[i][v] * x[i][v] : x[i][v];
                    b[v] = start ? u : fmaf(a[i][v], b[v], u);
                    A[v] = start ? 0.f : A[v] * a[i][v];
                }
            }
#pragma unroll
        for (int i = kSeg - 1; i >= 0; --i)
            if (i < n) {
                const bool start = (starts >> i) & 1u;
#pragma unroll
                for (int v = 0; v < V; ++v) send[v] = start ? 0.f : a[i][v] * (g[i][v] + send[v]);
            }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            sm.A[warp][lane * V + v] = A[v];
            sm.b[warp][lane * V + v] = b[v];
            back[warp][lane * V + v] = send[v];
        }
        if (lane == 0) sm.cut[warp] = starts != 0;
        __syncthreads();
        // 2. the state entering the segment; what comes to it from behind
#pragma unroll
        for (int j = 0; j < kWarps - 1; ++j)
            if (j < warp) {
                const bool cj = sm.cut[j] != 0;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float Aj = sm.A[j][lane * V + v], bj = sm.b[j][lane * V + v];
                    h[v] = cj ? bj : fmaf(Aj, h[v], bj);
                }
            }
        float qA[V], qb[V], from_behind[V];
        bool cut = false, own_cut = false;
#pragma unroll
        for (int v = 0; v < V; ++v) { qA[v] = 1.f; qb[v] = 0.f; }
#pragma unroll
        for (int j = kWarps - 1; j >= 0; --j) {
            if (j == warp) {
                own_cut = cut;
#pragma unroll
                for (int v = 0; v < V; ++v) { A[v] = qA[v]; from_behind[v] = qb[v]; }
            }
            const bool cj = sm.cut[j] != 0;
            cut |= cj;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float Aj = sm.A[j][lane * V + v], bj = back[j][lane * V + v];
                qb[v] = cj ? bj : fmaf(Aj, qb[v], bj);
                qA[v] = cj ? 0.f : Aj * qA[v];
            }
        }
        if (ranks > 1) {
            if (warp == 0) {
#pragma unroll
                for (int v = 0; v < V; ++v) { sm.cta_A[lane * V + v] = qA[v]; sm.cta_b[lane * V + v] = qb[v]; }
                if (lane == 0) sm.cta_cut = cut;
            }
            cluster.sync();
        }
        float e[V];
        for (int q = ranks - 1; q >= 0; --q) {
            const bool own = q == rank;
            const Summaries<V>* from = own ? &sm : cluster.map_shared_rank(&sm, q);
            const bool cq = own ? cut : from->cta_cut != 0;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float Aq = own ? qA[v] : from->cta_A[lane * V + v], bq = own ? qb[v] : from->cta_b[lane * V + v];
                if (own) e[v] = carry[v];
                carry[v] = cq ? bq : fmaf(Aq, carry[v], bq);
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) e[v] = own_cut ? from_behind[v] : fmaf(A[v], e[v], from_behind[v]);
        // 3. the states again, and in their place what df is dh times of; then back through the segment
#pragma unroll
        for (int i = 0; i < kSeg; ++i)
            if (i < n) {
                const bool start = (starts >> i) & 1u;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float before = start ? 0.f : h[v], xi = x[i][v];
                    const float u = kGate == kSigmoidGate ? w[i][v] * xi : xi;
                    h[v] = start ? u : fmaf(a[i][v], h[v], u);
                    x[i][v] = kGate == kSigmoidGate ? (before - xi) * a[i][v] * w[i][v] : start ? 0.f : -before * w[i][v];
                }
            }
#pragma unroll
        for (int i = kSeg - 1; i >= 0; --i)
            if (i < n) {
                const bool start = (starts >> i) & 1u;
                float ox[V], of[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float dh = g[i][v] + e[v];
                    ox[v] = kGate == kSigmoidGate ? dh * w[i][v] : dh;
                    of[v] = dh * x[i][v];
                    e[v] = start ? 0.f : a[i][v] * dh;
                }
                if (live) {
                    store_out<V>(dx + base + (size_t)(t0 + i) * p.C, ox);
                    store_out<V>(df + base + (size_t)(t0 + i) * p.C, of);
                }
            }
        if (tile == 0 && warp == 0 && live) {
#pragma unroll
            for (int v = 0; v < V; ++v) ds0[so + v] = e[v] + (L == 0 ? gstate[v] : 0.f);
        }
        if (ranks > 1) cluster.sync(); else __syncthreads();   // the summaries are read before the next ones are written
    }
}

// One token: out = h = (start ? 0 : a s) + u; rows of length 0 keep their state (and have their output all the same).  A thread's
// V channels are read before they are written, so s_out may be s.
template <typename T, int V, int kGate>
__global__ void __launch_bounds__(256)
gated_step_kernel(int B, int C, const T* x, long long x_stride, const T* f, long long f_stride, const float* s, long long s_stride,
                  const uint32_t* __restrict__ length, const uint8_t* __restrict__ starts, T* y, float* s_out, long long s_out_stride) {
    const int per_row = C / V;
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
    if (at >= (long long)B * per_row) return;
    const int bi = (int)(at / per_row), c = (int)(at - (long long)bi * per_row) * V;
    const bool start = starts != nullptr && starts[bi] != 0, keep = length != nullptr && length[bi] == 0;
    const Raw<T, V> rx = load_raw<T, V>(x + bi * x_stride + c), rf = load_raw<T, V>(f + bi * f_stride + c);
    const Raw<float, V> rs = load_raw<float, V>(s + bi * s_stride + c);
    float h[V], out[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float a, w;
        gate_of<T, kGate>(channel(rf, v), a, w);
        const float u = kGate == kSigmoidGate ? w * channel(rx, v) : channel(rx, v);
        out[v] = start ? u : fmaf(a, channel(rs, v), u);
        h[v] = keep ? channel(rs, v) : out[v];
    }
    store_out<V>(y + (size_t)bi * C + c, out);
    store_out<V>(s_out + bi * s_out_stride + c, h);
}

int cluster_size(int units, int tiles) {
    int n = 1;
    while (n < kMaxCluster && n < tiles && units * n < 2 * sm_count_of_current_device()) n *= 2;
    return n;
}
template <typename Kernel, typename... Args>
int launch(Kernel kern, cudaStream_t st, int B, const Problem& p, Args... args) {
    const int tiles = (p.T + kTile - 1) / kTile, ranks = cluster_size(B * p.slabs, tiles);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(B * p.slabs * ranks));
    cfg.blockDim = dim3(kWarps * 32);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, p, args...) == cudaSuccess ? B200WKV_OK : B200WKV_ELAUNCH;
}
// Two channels at a time where the rows allow it.
bool pairs(int C, size_t element, std::initializer_list<const void*> streams, std::initializer_list<const void*> states,
           std::initializer_list<long long> strides) {
    uintptr_t bits = 0, state_bits = 0;
    long long odd = C;
    for (const void* q : streams) bits |= reinterpret_cast<uintptr_t>(q);
    for (const void* q : states) state_bits |= reinterpret_cast<uintptr_t>(q);
    for (long long s : strides) odd |= s;
    return bits % (2 * element) == 0 && state_bits % 8 == 0 && odd % 2 == 0;
}

template <typename T, int V, int kGate>
int fwd(cudaStream_t st, int B, Problem p, void* y, float* s_out, float* ckpt) {
    p.slabs = (p.C + 32 * V - 1) / (32 * V);
    return launch(gated_fwd_kernel<T, V, kGate>, st, B, p, (T*)y, s_out, ckpt);
}
template <typename T, int V, int kGate>
int bwd(cudaStream_t st, int B, Problem p, const void* gy, const float* gs, const float* ckpt, void* dx, void* df, float* ds0) {
    p.slabs = (p.C + 32 * V - 1) / (32 * V);
    return launch(gated_bwd_kernel<T, V, kGate>, st, B, p, (const T*)gy, gs, ckpt, (T*)dx, (T*)df, ds0);
}
template <typename T, int V, int kGate>
int step(cudaStream_t st, int B, int C, const Stream& x, const Stream& f, const float* s, long long s_stride, const uint32_t* length,
         const uint8_t* starts, void* y, float* s_out, long long s_out_stride) {
    const long long threads = (long long)B * (C / V);
    gated_step_kernel<T, V, kGate><<<(unsigned)((threads + 255) / 256), 256, 0, st>>>(
        B, C, (const T*)x.p, x.batch, (const T*)f.p, f.batch, s, s_stride, length, starts, (T*)y, s_out, s_out_stride);
    return cudaGetLastError() == cudaSuccess ? B200WKV_OK : B200WKV_ELAUNCH;
}
// calls `go` with the element type, the channels at a time and the gate as template arguments
#define B200WKV_GATED(go, two, ...)                                                                                                  \
    (dtype == B200WKV_F32 ? (two ? (gate == B200WKV_GATE_SIGMOID ? go<float, 2, 0>(__VA_ARGS__) : go<float, 2, 1>(__VA_ARGS__))          \
                                 : (gate == B200WKV_GATE_SIGMOID ? go<float, 1, 0>(__VA_ARGS__) : go<float, 1, 1>(__VA_ARGS__)))         \
                          : (two ? (gate == B200WKV_GATE_SIGMOID ? go<__nv_bfloat16, 2, 0>(__VA_ARGS__) : go<__nv_bfloat16, 2, 1>(__VA_ARGS__)) \
                                 : (gate == B200WKV_GATE_SIGMOID ? go<__nv_bfloat16, 1, 0>(__VA_ARGS__) : go<__nv_bfloat16, 1, 1>(__VA_ARGS__))))
}  // namespace

size_t gated_residual_bytes(int B, int T, int C) { return (size_t)B * ((T + kTile - 1) / kTile) * C * sizeof(float); }

int gated_fwd(cudaStream_t st, int dtype, int gate, int B, int T, int C, const void* x, long long x_batch, long long x_token, const void* f,
              long long f_batch, long long f_token, const float* s0, const uint32_t* length, const uint8_t* ns, void* y, float* s_out,
              void* residual) {
    const Problem p = {T, C, 0, {x, x_batch, x_token}, {f, f_batch, f_token}, s0, length, ns};
    const bool two = pairs(C, dtype == B200WKV_F32 ? 4 : 2, {x, f, y}, {s0, s_out, residual}, {x_batch, x_token, f_batch, f_token});
    return B200WKV_GATED(fwd, two, st, B, p, y, s_out, (float*)residual);
}
int gated_bwd(cudaStream_t st, int dtype, int gate, int B, int T, int C, const void* x, long long x_batch, long long x_token, const void* f,
              long long f_batch, long long f_token, const uint32_t* length, const uint8_t* ns, const void* gy, const float* gs,
              const void* residual, void* dx, void* df, float* ds0) {
    const Problem p = {T, C, 0, {x, x_batch, x_token}, {f, f_batch, f_token}, nullptr, length, ns};
    const bool two = pairs(C, dtype == B200WKV_F32 ? 4 : 2, {x, f, gy, dx, df}, {gs, residual, ds0}, {x_batch, x_token, f_batch, f_token});
    return B200WKV_GATED(bwd, two, st, B, p, gy, gs, (const float*)residual, dx, df, ds0);
}
int gated_step(cudaStream_t st, int dtype, int gate, int B, int C, const void* x, long long x_stride, const void* f, long long f_stride,
               const float* s, long long s_stride, const uint32_t* length, const uint8_t* ns, void* y, float* s_out, long long s_out_stride) {
    const bool two = pairs(C, dtype == B200WKV_F32 ? 4 : 2, {x, f, y}, {s, s_out}, {x_stride, f_stride, s_stride, s_out_stride});
    const Stream sx = {x, x_stride, 0}, sf = {f, f_stride, 0};
    return B200WKV_GATED(step, two, st, B, C, sx, sf, s, s_stride, length, ns, y, s_out, s_out_stride);
}

}  // namespace b200wkv
