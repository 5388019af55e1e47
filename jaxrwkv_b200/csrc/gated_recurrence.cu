// Gated linear recurrence, one number of state per channel, fp32 arithmetic and state:
//   gate "sigmoid":  a = sigmoid(f)      u = (1 - a) x
//   gate "decay":    a = exp(-exp(f))    u = x             (f: the raw log-log decay, as RWKV-7's w)
//   h_t = (start_t ? 0 : a_t h_{t-1}) + u_t     out_t = h_t     s_out = h_{length-1}
// Both gates lie in [0, 1], so a product of them over any stretch of tokens cannot overflow.
//
// The recurrence is associative: a stretch of tokens acts on the state entering it as h -> A h + b.  A CTA of eight warps owns
// 64 channels of one sequence, a pair a lane, each warp consecutive segments of tokens, and the CTAs of a cluster own
// consecutive tiles in turn:
//   1. every warp turns its segment, which cp.async has brought into shared memory rounds ago, into gates and increments in
//      registers, asks for the segment two rounds on, and reduces what it has to (A, b);
//   2. the warps' (A, b) are combined in order through shared memory; where a cluster shares the sequence, the last warp sends
//      the whole tile's to every CTA of it (st.async onto an mbarrier there), and everyone carries the state over all tiles of
//      the round: one hop, whatever the size of the cluster;
//   3. every warp walks its segment from the state that enters it and writes the outputs.
//
// Backward: dh_t = gy_t + [t == length-1] gs + c_{t+1},  c_t = start_t ? 0 : a_t dh_t.  The states are recomputed from the
// state entering each tile of 64 tokens, which the forward keeps (4 bytes per 64 tokens and channel); c runs over the segments
// from the last to the first with the same products A.
//
// A start flag cuts by a select, not by a factor of 0: what is no number in front of it ends there.
#include <limits.h>

#include <initializer_list>

#include "common.cuh"
#include "device_once.cuh"
#include "gate_math.cuh"
#include "host_calls.h"
#include "tc05.cuh"

namespace b200wkv {
int* wkv7_chunk_status_word();
namespace {
using namespace tc;

constexpr int kWarps = 8;
constexpr int kWide = 64;                  // channels of a CTA
constexpr int kKept = 64;                  // tokens per kept state, and of a backward tile
constexpr int kMaxCluster = 8;
constexpr int kStages = 2;
constexpr int kWaitRanOut = 3;             // status word: a wait for the other CTAs of a cluster

// two channels, as they lie in shared memory
__device__ __forceinline__ float2 pair_at(const float* p) { return *reinterpret_cast<const float2*>(p); }
__device__ __forceinline__ float2 pair_at(const __nv_bfloat16* p) { return unpack_pair(*reinterpret_cast<const uint32_t*>(p)); }
__device__ __forceinline__ void store_pair(float* p, float a, float b) { *reinterpret_cast<float2*>(p) = make_float2(a, b); }
__device__ __forceinline__ void store_pair(__nv_bfloat16* p, float a, float b) { *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b); }

constexpr int kSigmoidGate = B200WKV_GATE_SIGMOID;
// The gate a, and what the backward needs of it: `w`, for the sigmoid 1 - a (to full relative precision), for the decay -da/df.
template <typename T, int kGate> __device__ __forceinline__ void gate_of(float2 f, float2& a, float2& w) {
    if (kGate == kSigmoidGate) {
        sigmoid_pair<T>(f, a, w);
    } else {
        // (accurate in 16 bits too: the state sums 1 / (1 - a) tokens, and an error of a is that much larger in it)
        const float2 e = make_float2(expf(f.x), expf(f.y));
        a = make_float2(expf(-e.x), expf(-e.y));
        w = mul2(e, a);
        w = make_float2(a.x == 0.f ? 0.f : w.x, a.y == 0.f ? 0.f : w.y);        // (e may be infinite then)
    }
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
    int* status;
};

// What a stretch does to the state of a channel: h -> A h + b.  A's sign bit says that a start flag lies inside: h is dropped.
__device__ __forceinline__ bool cuts(float A) { return __float_as_int(A) < 0; }
__device__ __forceinline__ float behind(float A, float b, float h) { return cuts(A) ? b : fmaf(A, h, b); }
struct Stretch {
    float4 v;                              // A, b of the lane's first channel, then of its second
    __device__ __forceinline__ static Stretch nothing() { return {make_float4(1.f, 0.f, 1.f, 0.f)}; }
    __device__ __forceinline__ void follow(float4 n) {               // by the stretch n
        v.y = behind(n.x, n.y, v.y);
        v.w = behind(n.z, n.w, v.w);
        v.x = cuts(n.x) ? -1.f : v.x * n.x;
        v.z = cuts(n.z) ? -1.f : v.z * n.z;
    }
    __device__ __forceinline__ float2 of(float2 h) const { return make_float2(behind(v.x, v.y, h.x), behind(v.z, v.w, h.y)); }
};

// A warp's segments of one stream on their way to shared memory: kSeg rows of 64 channels, zeros behind the sequence's end and the
// last channel.  Pieces of kPiece bytes; 2: single 16-bit elements, which no asynchronous copy takes.
template <typename T, int kPiece, int kSeg> struct Feed {
    static constexpr int kPer = kPiece / (int)sizeof(T), kPerRow = kWide / kPer;
    static constexpr int kRows = kPerRow <= 32 ? 32 / kPerRow : 1, kPasses = kPerRow <= 32 ? 1 : kPerRow / 32;
    const T* from;                         // the lane's first piece of token 0
    long long stride;
    int row, c, left;                      // the lane's first row and channel; channels that there are
    __device__ __forceinline__ Feed(const void* p, long long batch, long long token, int bi, int c0, int C, int lane)
        : stride(token), row(kPasses == 1 ? lane / kPerRow : 0), c((kPasses == 1 ? lane % kPerRow : lane) * kPer), left(C - c0) {
        from = (const T*)p + bi * batch + c0;
    }
    __device__ __forceinline__ static void piece(T* to, const T* from, bool valid) {
        if constexpr (kPiece == 16) cp_async16(to, from, valid);
        else if constexpr (kPiece == 4)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(valid ? 4 : 0) : "memory");
        else *to = valid ? *from : from_f32<T>(0.f);
    }
    __device__ __forceinline__ void fetch(T* to, int t0, int Tlen) const {
        to += row * kWide + c;
        if (t0 + kSeg <= Tlen && left >= kWide) {
            const T* at = from + (t0 + row) * stride + c;
#pragma unroll
            for (int i = 0; i < kSeg; i += kRows, at += kRows * stride)
#pragma unroll
                for (int pass = 0; pass < kPasses; ++pass) piece(to + i * kWide + pass * 32 * kPer, at + pass * 32 * kPer, true);
        } else {
#pragma unroll
            for (int i = 0; i < kSeg; i += kRows)
#pragma unroll
                for (int pass = 0; pass < kPasses; ++pass) {
                    const int t = t0 + i + row, ch = c + pass * 32 * kPer;
                    const bool valid = t < Tlen && ch < left;
                    piece(to + i * kWide + pass * 32 * kPer, from + (valid ? t * stride + ch : 0), valid);
                }
        }
    }
};
__device__ __forceinline__ void fetched() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void wait_fetched() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
    __syncwarp();
}

// A pair of channels of a dense row; single elements where pairs do not fit the row (kPiece one element) or its end
template <typename T, int kPiece> __device__ __forceinline__ void put(T* p, float a, float b, int channels) {
    if constexpr (kPiece >= 2 * (int)sizeof(T)) {
        if (channels > 0) store_pair(p, a, b);
    } else {
        if (channels > 0) p[0] = from_f32<T>(a);
        if (channels > 1) p[1] = from_f32<T>(b);
    }
}
__device__ __forceinline__ float2 get_state(const float* p, int channels) {
    return make_float2(p != nullptr && channels > 0 ? p[0] : 0.f, p != nullptr && channels > 1 ? p[1] : 0.f);
}
__device__ __forceinline__ void put_state(float* p, float2 h, int channels) {
    if (channels > 0) p[0] = h.x;
    if (channels > 1) p[1] = h.y;
}

// start flags of the kSeg tokens from t0 on as a bit mask (bit i = token t0 + i)
template <int kSeg> __device__ __forceinline__ uint32_t segment_flags(const uint8_t* ns, int t0, int Tlen, int lane) {
    if (ns == nullptr) return 0;
    return __ballot_sync(0xffffffffu, lane < kSeg && t0 + lane < Tlen && ns[t0 + lane] != 0);
}

// What the CTAs of a cluster tell one another: the stretches of a round's tiles.  Two rounds' worth: a CTA sends a round's only when
// it has those of the round in front from everyone, who by then have used the round before that.
struct Exchange {
    float4 tiles[2][kMaxCluster][32];
    uint64_t bar[2];
    __device__ __forceinline__ void open(int ranks) {
        if (threadIdx.x == 0) {
            mbar_init(&bar[0], 1);
            mbar_init(&bar[1], 1);
            mbar_init_fence();
        }
        if (ranks > 1) cluster_sync();
    }
    __device__ __forceinline__ void send(int round, int rank, int ranks, const Stretch& tile, int lane) {   // by one warp
        uint64_t* const mine = &bar[round & 1];
        if (lane == 0) mbar_expect_tx(mine, (uint32_t)ranks * 32 * sizeof(float4));
        for (int q = 0; q < ranks; ++q) store_in_cta(in_cta(&tiles[round & 1][rank][lane], q), tile.v, in_cta(mine, q));
    }
    __device__ __forceinline__ void wait(int round, bool& lost, int* status) {
        if (lost || mbar_wait_cluster(&bar[round & 1], (round >> 1) & 1)) return;
        lost = true;
        if (status != nullptr) *status = kWaitRanOut;
    }
    // no CTA leaves while others may still send to it
    __device__ __forceinline__ void close(int ranks) { if (ranks > 1) cluster_sync(); }
};

struct Place {
    int rank, ranks, lane, warp, bi, c, channels, L;
    size_t state;                          // the lane's first channel in a dense (B, C) array
    __device__ __forceinline__ Place(const Problem& p) {
        rank = (int)cluster_rank(); ranks = (int)cluster_size();
        lane = threadIdx.x & 31; warp = threadIdx.x >> 5;
        const int unit = blockIdx.x / ranks;
        bi = unit / p.slabs;
        c = unit % p.slabs * kWide + 2 * lane;
        channels = p.C - c;
        L = p.length != nullptr ? (int)min(p.length[bi], (uint32_t)p.T) : p.T;
        state = (size_t)bi * p.C + c;
    }
};
struct Plain { static constexpr bool value = true; };      // a whole segment without a start flag in which the returned state is not taken
struct Marked { static constexpr bool value = false; };

template <typename T> constexpr int kFwdSeg = sizeof(T) == 2 ? 16 : 8;
constexpr int kBwdSeg = kKept / kWarps;

template <typename T, int kGate, int kPiece>
__global__ void __launch_bounds__(kWarps * 32, 2)
gated_fwd_kernel(const Problem p, T* __restrict__ y, float* __restrict__ s_out, float* __restrict__ kept) {
    constexpr int kSeg = kFwdSeg<T>, kTile = kSeg * kWarps, kHalf = kSeg * kWide;
    extern __shared__ __align__(128) unsigned char dynamic[];
    __shared__ Exchange ex;
    __shared__ float4 segs[2][kWarps][32];
    __shared__ float2 carried[2][32];
    const Place at(p);
    const int lane = at.lane, warp = at.warp, ranks = at.ranks, tiles = (p.T + kTile - 1) / kTile, rounds = (tiles + ranks - 1) / ranks;
    const Feed<T, kPiece, kSeg> fx(p.x.p, p.x.batch, p.x.token, at.bi, at.c - 2 * lane, p.C, lane);
    const Feed<T, kPiece, kSeg> ff(p.f.p, p.f.batch, p.f.token, at.bi, at.c - 2 * lane, p.C, lane);
    T* const room = (T*)dynamic + warp * kStages * 2 * kHalf;
    const auto first = [&](int round) { return (round * ranks + at.rank) * kTile + warp * kSeg; };
    const auto ask = [&](int round) {
        if (round < rounds) {
            T* const to = room + round % kStages * 2 * kHalf;
            fx.fetch(to, first(round), p.T);
            ff.fetch(to + kHalf, first(round), p.T);
        }
        fetched();
    };
    for (int i = 0; i < kStages; ++i) ask(i);
    float2 carry = get_state(p.s0 != nullptr ? p.s0 + at.state : nullptr, at.channels);      // state entering the round
    if (at.L == 0 && warp == 0 && at.rank == 0) put_state(s_out + at.state, carry, at.channels);
    if (warp == kWarps - 1) carried[0][lane] = carry;
    ex.open(ranks);
    bool lost = false;
    T* const py = y + (size_t)at.bi * p.T * p.C + at.c;
    const uint8_t* const ns = p.starts != nullptr ? p.starts + (size_t)at.bi * p.T : nullptr;
    for (int round = 0; round < rounds; ++round) {
        const int t0 = first(round), n = max(0, min(kSeg, p.T - t0)), parity = round & 1;
        const uint32_t starts = segment_flags<kSeg>(ns, t0, p.T, lane);
        const bool plain = n == kSeg && starts == 0 && (at.L <= t0 || at.L > t0 + kSeg);
        // 1. gates and increments, and what the segment does
        float2 a[kSeg], u[kSeg];
        wait_fetched<kStages - 1>();
        const T* const from = room + round % kStages * 2 * kHalf + 2 * lane;
#pragma unroll
        for (int i = 0; i < kSeg; ++i) {
            const float2 x = pair_at(from + i * kWide);
            float2 w;
            gate_of<T, kGate>(pair_at(from + kHalf + i * kWide), a[i], w);
            u[i] = kGate == kSigmoidGate ? mul2(w, x) : x;
        }
        __syncwarp();                      // the segment has been read
        ask(round + kStages);
        float2 A = both(1.f), b = both(0.f);
        const auto summarise = [&](auto kind) {
#pragma unroll
            for (int i = 0; i < kSeg; ++i) {
                if (!kind.value) {
                    if (i >= n) { a[i] = both(1.f); u[i] = both(0.f); }
                    if ((starts >> i) & 1u) { A = both(-1.f); b = u[i]; continue; }
                }
                b = fma2(a[i], b, u[i]);
                A = mul2(A, a[i]);
            }
        };
        if (plain) summarise(Plain()); else summarise(Marked());
        const Stretch own = {make_float4(A.x, b.x, A.y, b.y)};
        segs[parity][warp][lane] = own.v;
        __syncthreads();
        // 2. the state that enters the segment
        float2 h;
        if (ranks > 1) {
            Stretch front = Stretch::nothing();
#pragma unroll
            for (int j = 0; j < kWarps - 1; ++j)
                if (j < warp) front.follow(segs[parity][j][lane]);
            if (warp == kWarps - 1) {
                Stretch tile = front;
                tile.follow(own.v);
                ex.send(round, at.rank, ranks, tile, lane);
            }
            ex.wait(round, lost, p.status);
            for (int q = 0; q < ranks; ++q) {
                if (q == at.rank) h = carry;
                const Stretch tile = {ex.tiles[parity][q][lane]};
                carry = tile.of(carry);
            }
            h = front.of(h);
        } else {
            h = carried[parity][lane];
#pragma unroll
            for (int j = 0; j < kWarps - 1; ++j)
                if (j < warp) h = Stretch{segs[parity][j][lane]}.of(h);
        }
        // (a kept state is wanted in front of every 64th token; the returned one behind its token)
        if (kept != nullptr && n > 0 && t0 % kKept == 0) put_state(kept + ((size_t)at.bi * ((p.T + kKept - 1) / kKept) + t0 / kKept) * p.C + at.c, h, at.channels);
        // 3. outputs
        T* to = py + (size_t)t0 * p.C;
        const auto walk = [&](auto kind) {
#pragma unroll
            for (int i = 0; i < kSeg; ++i, to += p.C) {
                const bool start = !kind.value && ((starts >> i) & 1u);
                h = start ? u[i] : fma2(a[i], h, u[i]);
                if (kind.value || i < n) put<T, kPiece>(to, h.x, h.y, at.channels);
                if (!kind.value && t0 + i == at.L - 1) put_state(s_out + at.state, h, at.channels);
            }
        };
        if (plain) walk(Plain()); else walk(Marked());
        if (ranks == 1 && warp == kWarps - 1) carried[parity ^ 1][lane] = h;
    }
    ex.close(ranks);
}

template <typename T, int kGate, int kPiece>
__global__ void __launch_bounds__(kWarps * 32, 2)
gated_bwd_kernel(const Problem p, const T* __restrict__ gy, const float* __restrict__ gs, const float* __restrict__ kept,
                 T* __restrict__ dx, T* __restrict__ df, float* __restrict__ ds0) {
    constexpr int kSeg = kBwdSeg, kTile = kKept, kHalf = kSeg * kWide;
    extern __shared__ __align__(128) unsigned char dynamic[];
    __shared__ Exchange ex;
    __shared__ float4 segs[2][kWarps][32];
    __shared__ float2 sent[2][kWarps][32], carried[2][32];
    const Place at(p);
    const int lane = at.lane, warp = at.warp, ranks = at.ranks, tiles = (p.T + kTile - 1) / kTile, rounds = (tiles + ranks - 1) / ranks;
    const Feed<T, kPiece, kSeg> fx(p.x.p, p.x.batch, p.x.token, at.bi, at.c - 2 * lane, p.C, lane);
    const Feed<T, kPiece, kSeg> ff(p.f.p, p.f.batch, p.f.token, at.bi, at.c - 2 * lane, p.C, lane);
    const Feed<T, kPiece, kSeg> fg(gy, (long long)p.T * p.C, p.C, at.bi, at.c - 2 * lane, p.C, lane);
    T* const room = (T*)dynamic + warp * kStages * 3 * kHalf;
    // rounds are taken from the last to the first; `done` of them lie behind
    const auto first = [&](int done) { return ((rounds - 1 - done) * ranks + at.rank) * kTile + warp * kSeg; };
    const auto ask = [&](int done) {
        if (done < rounds) {
            T* const to = room + done % kStages * 3 * kHalf;
            fx.fetch(to, first(done), p.T);
            ff.fetch(to + kHalf, first(done), p.T);
            if (gy != nullptr) fg.fetch(to + 2 * kHalf, first(done), p.T);
        }
        fetched();
    };
    const auto entering = [&](int done) {  // the kept state in front of a round's tile
        const int tile = (rounds - 1 - done) * ranks + at.rank;
        return done < rounds && tile < tiles ? get_state(kept + ((size_t)at.bi * tiles + tile) * p.C + at.c, at.channels) : make_float2(0.f, 0.f);
    };
    for (int i = 0; i < kStages; ++i) ask(i);
    float2 next = entering(0), carry = make_float2(0.f, 0.f);      // carry: c entering the round from behind
    const float2 gstate = get_state(gs != nullptr ? gs + at.state : nullptr, at.channels);
    if (warp == 0) carried[0][lane] = carry;
    ex.open(ranks);
    bool lost = false;
    const size_t base = (size_t)at.bi * p.T * p.C + at.c;
    const uint8_t* const ns = p.starts != nullptr ? p.starts + (size_t)at.bi * p.T : nullptr;
    for (int done = 0; done < rounds; ++done) {
        const int t0 = first(done), n = max(0, min(kSeg, p.T - t0)), parity = done & 1;
        const uint32_t starts = segment_flags<kSeg>(ns, t0, p.T, lane);
        const bool plain = n == kSeg && starts == 0 && (at.L <= t0 || at.L > t0 + kSeg);
        float2 h = next;
        next = entering(done + 1);
        // 1. gates; what the segment does to the states, and what it sends to the front
        float2 a[kSeg], w[kSeg], x[kSeg], g[kSeg];
        wait_fetched<kStages - 1>();
        const T* const from = room + done % kStages * 3 * kHalf + 2 * lane;
#pragma unroll
        for (int i = 0; i < kSeg; ++i) {
            x[i] = pair_at(from + i * kWide);
            gate_of<T, kGate>(pair_at(from + kHalf + i * kWide), a[i], w[i]);
            g[i] = gy != nullptr ? pair_at(from + 2 * kHalf + i * kWide) : both(0.f);
        }
        __syncwarp();                      // the segment has been read
        ask(done + kStages);
        const auto increment = [&](int i) { return kGate == kSigmoidGate ? mul2(w[i], x[i]) : x[i]; };
        float2 A = both(1.f), b = both(0.f), c = both(0.f);
        const auto summarise = [&](auto kind) {
#pragma unroll
            for (int i = 0; i < kSeg; ++i) {
                if (!kind.value) {
                    if (i >= n) { a[i] = both(1.f); w[i] = x[i] = both(0.f); }
                    if (t0 + i == at.L - 1) g[i] = add2(g[i], gstate);
                    if ((starts >> i) & 1u) { A = both(-1.f); b = increment(i); continue; }
                }
                b = fma2(a[i], b, increment(i));
                A = mul2(A, a[i]);
            }
#pragma unroll
            for (int i = kSeg - 1; i >= 0; --i) c = !kind.value && ((starts >> i) & 1u) ? both(0.f) : mul2(a[i], add2(g[i], c));
        };
        if (plain) summarise(Plain()); else summarise(Marked());
        const Stretch own = {make_float4(A.x, b.x, A.y, b.y)};
        segs[parity][warp][lane] = own.v;
        sent[parity][warp][lane] = c;
        __syncthreads();
        // 2. the state that enters the segment, and c that enters it from behind
#pragma unroll
        for (int j = 0; j < kWarps - 1; ++j)
            if (j < warp) h = Stretch{segs[parity][j][lane]}.of(h);
        const auto before = [&](int j) {
            const float4 s = segs[parity][j][lane];
            const float2 b = sent[parity][j][lane];
            return make_float4(s.x, b.x, s.z, b.y);
        };
        float2 e;
        if (ranks > 1) {
            Stretch rear = Stretch::nothing();
#pragma unroll
            for (int j = kWarps - 1; j > 0; --j)
                if (j > warp) rear.follow(before(j));
            if (warp == 0) {
                Stretch tile = rear;
                tile.follow(make_float4(own.v.x, c.x, own.v.z, c.y));
                ex.send(done, at.rank, ranks, tile, lane);
            }
            ex.wait(done, lost, p.status);
            for (int q = ranks - 1; q >= 0; --q) {
                if (q == at.rank) e = carry;
                const Stretch tile = {ex.tiles[parity][q][lane]};
                carry = tile.of(carry);
            }
            e = rear.of(e);
        } else {
            e = carried[parity][lane];
#pragma unroll
            for (int j = kWarps - 1; j > 0; --j)
                if (j > warp) e = Stretch{before(j)}.of(e);
        }
        // 3. the states again, and in the place of x what df is dx times of; then back through the segment
        const auto walk = [&](auto kind) {
#pragma unroll
            for (int i = 0; i < kSeg; ++i) {
                const bool start = !kind.value && ((starts >> i) & 1u);
                const float2 in = start ? both(0.f) : h, u = increment(i);
                h = start ? u : fma2(a[i], h, u);
                if (kGate == kSigmoidGate) x[i] = mul2(fma2(x[i], both(-1.f), in), a[i]);
                else x[i] = start ? both(0.f) : mul2(mul2(in, w[i]), both(-1.f));
            }
            const size_t last = base + (size_t)(t0 + kSeg - 1) * p.C;
            T *to_x = dx + last, *to_f = df + last;
#pragma unroll
            for (int i = kSeg - 1; i >= 0; --i, to_x -= p.C, to_f -= p.C) {
                const float2 d = add2(g[i], e), o = kGate == kSigmoidGate ? mul2(d, w[i]) : d, of = mul2(o, x[i]);
                if (kind.value || i < n) {
                    put<T, kPiece>(to_x, o.x, o.y, at.channels);
                    put<T, kPiece>(to_f, of.x, of.y, at.channels);
                }
                e = !kind.value && ((starts >> i) & 1u) ? both(0.f) : mul2(a[i], d);
            }
        };
        if (plain) walk(Plain()); else walk(Marked());
        if (t0 == 0) put_state(ds0 + at.state, at.L == 0 ? make_float2(e.x + gstate.x, e.y + gstate.y) : e, at.channels);
        if (ranks == 1 && warp == 0) carried[parity ^ 1][lane] = e;
    }
    ex.close(ranks);
}

// One token: out = h = (start ? 0 : a s) + u; rows of length 0 keep their state (and have their output all the same).  A thread's
// V channels are read before they are written, so s_out may be s.
template <typename T, int V> struct alignas(V * sizeof(T) < 16 ? V * sizeof(T) : 16) Few { T q[V]; };
template <typename T, int V, int kGate>
__global__ void __launch_bounds__(256)
gated_step_kernel(int B, int C, const T* x, long long x_stride, const T* f, long long f_stride, const float* s, long long s_stride,
                  const uint32_t* __restrict__ length, const uint8_t* __restrict__ starts, T* y, float* s_out, long long s_out_stride) {
    const int per_row = C / V;
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
    if (at >= (long long)B * per_row) return;
    const int bi = (int)(at / per_row), c = (int)(at - (long long)bi * per_row) * V;
    const bool start = starts != nullptr && starts[bi] != 0, keep = length != nullptr && length[bi] == 0;
    const Few<T, V> rx = *(const Few<T, V>*)(x + bi * x_stride + c), rf = *(const Few<T, V>*)(f + bi * f_stride + c);
    const Few<float, V> rs = *(const Few<float, V>*)(s + bi * s_stride + c);
    Few<T, V> ry;
    Few<float, V> rh;
#pragma unroll
    for (int v = 0; v < V; v += 2) {
        const int v1 = v + (V > 1);        // (one channel: twice the same)
        const float2 x2 = make_float2(to_f32(rx.q[v]), to_f32(rx.q[v1])), s2 = make_float2(rs.q[v], rs.q[v1]);
        float2 a, w;
        gate_of<T, kGate>(make_float2(to_f32(rf.q[v]), to_f32(rf.q[v1])), a, w);
        const float2 u = kGate == kSigmoidGate ? mul2(w, x2) : x2, out = start ? u : fma2(a, s2, u);
        ry.q[v] = from_f32<T>(out.x);
        ry.q[v1] = from_f32<T>(out.y);
        rh.q[v] = keep ? s2.x : out.x;
        rh.q[v1] = keep ? s2.y : out.y;
    }
    *(Few<T, V>*)(y + (size_t)bi * C + c) = ry;
    *(Few<float, V>*)(s_out + bi * s_out_stride + c) = rh;
}

// How many clusters of n CTAs a kernel has on the device at a time, asked once per device and kernel (which sets its shared memory too).
struct Residency {
    DeviceOnce once;
    int clusters[kMaxDevices][kMaxCluster + 1];
    template <typename Kernel> const int* of(Kernel kern, size_t smem) {
        const int dev = current_device();
        if (dev < 0) return nullptr;
        const bool ok = once.ok([&]() {
            const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
            for (int n = 1; n <= kMaxCluster; ++n) {
                cudaLaunchAttribute attr[1];
                cudaLaunchConfig_t cfg = config(attr, n, n, smem, nullptr);
                int fit = 0;
                if (cudaOccupancyMaxActiveClusters(&fit, kern, &cfg) != cudaSuccess) {
                    (void)cudaGetLastError();
                    fit = 0;               // no cluster of this size
                }
                clusters[dev][n] = fit;
            }
            return e;
        });
        return ok ? clusters[dev] : nullptr;
    }
    static cudaLaunchConfig_t config(cudaLaunchAttribute* attr, int ranks, unsigned grid, size_t smem, cudaStream_t st) {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = ranks; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(grid);
        cfg.blockDim = dim3(kWarps * 32);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        return cfg;
    }
};
// CTAs of a cluster: those with which the last sequence is done after the fewest rounds, waves of clusters counted; the smaller of equals.
// units: 64 channels of a sequence each; tiles: of one of them.
int ranks_of(const int* resident, long long units, int tiles) {
    int best = 1;
    long long least = LLONG_MAX;
    for (int n = 1; n <= kMaxCluster && n <= tiles; ++n) {
        if (resident[n] < 1) continue;
        const long long rounds = (units + resident[n] - 1) / resident[n] * ((tiles + n - 1) / n);
        if (rounds < least) { least = rounds; best = n; }
    }
    return best;
}
template <typename Kernel, typename... Args>
int launch(Residency& residency, Kernel kern, cudaStream_t st, int B, const Problem& p, int tile, size_t smem, Args... args) {
    const int* const resident = residency.of(kern, smem);
    if (resident == nullptr) return B200WKV_ELAUNCH;
    const int units = B * p.slabs, ranks = ranks_of(resident, units, (p.T + tile - 1) / tile);
    cudaLaunchAttribute attr[1];
    const cudaLaunchConfig_t cfg = Residency::config(attr, ranks, (unsigned)units * ranks, smem, st);
    return cudaLaunchKernelEx(&cfg, kern, p, args...) == cudaSuccess ? B200WKV_OK : B200WKV_ELAUNCH;
}
// The widest pieces that every row of these begins on.
int piece_of(int C, int element, std::initializer_list<const void*> streams, std::initializer_list<long long> strides) {
    uintptr_t bits = (uintptr_t)C * element;
    for (const void* q : streams) bits |= reinterpret_cast<uintptr_t>(q);
    for (long long s : strides) bits |= (uintptr_t)s * element;
    return bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 2;
}

template <typename T, int kGate, int kPiece> int fwd(cudaStream_t st, int B, const Problem& p, void* y, float* s_out, float* kept) {
    static Residency once;
    constexpr int kTile = kFwdSeg<T> * kWarps;
    return launch(once, gated_fwd_kernel<T, kGate, kPiece>, st, B, p, kTile, (size_t)kStages * 2 * kTile * kWide * sizeof(T), (T*)y, s_out, kept);
}
template <typename T, int kGate, int kPiece>
int bwd(cudaStream_t st, int B, const Problem& p, const void* gy, const float* gs, const float* kept, void* dx, void* df, float* ds0) {
    static Residency once;
    return launch(once, gated_bwd_kernel<T, kGate, kPiece>, st, B, p, kKept, (size_t)kStages * 3 * kKept * kWide * sizeof(T), (const T*)gy, gs, kept,
                  (T*)dx, (T*)df, ds0);
}
// calls `go` with the element type, the gate and the piece as template arguments
#define B200WKV_GATED_PIECE(go, T, piece, ...) \
    (piece == 16 ? B200WKV_GATED_GATE(go, T, 16, __VA_ARGS__) : piece == 4 ? B200WKV_GATED_GATE(go, T, 4, __VA_ARGS__) : B200WKV_GATED_GATE(go, T, (int)sizeof(T), __VA_ARGS__))
#define B200WKV_GATED_GATE(go, T, n, ...) (gate == B200WKV_GATE_SIGMOID ? go<T, 0, n>(__VA_ARGS__) : go<T, 1, n>(__VA_ARGS__))

template <typename T, int V, int kGate>
int step(cudaStream_t st, int B, int C, const Stream& x, const Stream& f, const float* s, long long s_stride, const uint32_t* length,
         const uint8_t* starts, void* y, float* s_out, long long s_out_stride) {
    const long long threads = (long long)B * (C / V);
    gated_step_kernel<T, V, kGate><<<(unsigned)((threads + 255) / 256), 256, 0, st>>>(
        B, C, (const T*)x.p, x.batch, (const T*)f.p, f.batch, s, s_stride, length, starts, (T*)y, s_out, s_out_stride);
    return cudaGetLastError() == cudaSuccess ? B200WKV_OK : B200WKV_ELAUNCH;
}
}  // namespace

size_t gated_residual_bytes(int B, int T, int C) { return (size_t)B * ((T + kKept - 1) / kKept) * C * sizeof(float); }

int gated_fwd(cudaStream_t st, int dtype, int gate, int B, int T, int C, const void* x, long long x_batch, long long x_token, const void* f,
              long long f_batch, long long f_token, const float* s0, const uint32_t* length, const uint8_t* ns, void* y, float* s_out,
              void* residual) {
    const Problem p = {T, C, (C + kWide - 1) / kWide, {x, x_batch, x_token}, {f, f_batch, f_token}, s0, length, ns, wkv7_chunk_status_word()};
    const int piece = piece_of(C, dtype == B200WKV_F32 ? 4 : 2, {x, f, y}, {x_batch, x_token, f_batch, f_token});
    return dtype == B200WKV_F32 ? B200WKV_GATED_PIECE(fwd, float, piece, st, B, p, y, s_out, (float*)residual)
                                : B200WKV_GATED_PIECE(fwd, __nv_bfloat16, piece, st, B, p, y, s_out, (float*)residual);
}
int gated_bwd(cudaStream_t st, int dtype, int gate, int B, int T, int C, const void* x, long long x_batch, long long x_token, const void* f,
              long long f_batch, long long f_token, const uint32_t* length, const uint8_t* ns, const void* gy, const float* gs,
              const void* residual, void* dx, void* df, float* ds0) {
    const Problem p = {T, C, (C + kWide - 1) / kWide, {x, x_batch, x_token}, {f, f_batch, f_token}, nullptr, length, ns, wkv7_chunk_status_word()};
    const int piece = piece_of(C, dtype == B200WKV_F32 ? 4 : 2, {x, f, gy, dx, df}, {x_batch, x_token, f_batch, f_token});
    return dtype == B200WKV_F32 ? B200WKV_GATED_PIECE(bwd, float, piece, st, B, p, gy, gs, (const float*)residual, dx, df, ds0)
                                : B200WKV_GATED_PIECE(bwd, __nv_bfloat16, piece, st, B, p, gy, gs, (const float*)residual, dx, df, ds0);
}
int gated_step(cudaStream_t st, int dtype, int gate, int B, int C, const void* x, long long x_stride, const void* f, long long f_stride,
               const float* s, long long s_stride, const uint32_t* length, const uint8_t* ns, void* y, float* s_out, long long s_out_stride) {
    const Stream sx = {x, x_stride, 0}, sf = {f, f_stride, 0};
    // four channels a thread where rows and addresses allow it
    uintptr_t bits = (uintptr_t)C | (uintptr_t)x_stride | (uintptr_t)f_stride | (uintptr_t)s_stride | (uintptr_t)s_out_stride;
    const size_t few = 4 * (dtype == B200WKV_F32 ? 4 : 2);
    const bool four = bits % 4 == 0 && (uintptr_t)x % few == 0 && (uintptr_t)f % few == 0 && (uintptr_t)y % few == 0 && (uintptr_t)s % 16 == 0 &&
                      (uintptr_t)s_out % 16 == 0;
    const auto go = [&](auto fn) { return fn(st, B, C, sx, sf, s, s_stride, length, ns, y, s_out, s_out_stride); };
    const bool sigmoid = gate == B200WKV_GATE_SIGMOID;
    if (dtype == B200WKV_F32) return four ? (sigmoid ? go(step<float, 4, 0>) : go(step<float, 4, 1>)) : (sigmoid ? go(step<float, 1, 0>) : go(step<float, 1, 1>));
    return four ? (sigmoid ? go(step<__nv_bfloat16, 4, 0>) : go(step<__nv_bfloat16, 4, 1>))
                : (sigmoid ? go(step<__nv_bfloat16, 1, 0>) : go(step<__nv_bfloat16, 1, 1>));
}

}  // namespace b200wkv
