// Gated linear recurrence, one number of state per channel, fp32 arithmetic and state:
//   gate "sigmoid":  a = sigmoid(f)      u = (1 - a) x
//   gate "decay":    a = exp(-exp(f))    u = x             (f: the raw log-log decay, as RWKV-7's w)
//   h_t = (start_t ? 0 : a_t h_{t-1}) + u_t     out_t = h_t     s_out = h_{length-1}
// Both gates lie in [0, 1], so a product of them over any stretch of tokens cannot overflow.
//
// Memory bounds it: 3 elements a token and channel forward, 5 backward, and the kept states.  A CTA of eight warps owns 64 channels of one
// sequence, two a lane, and its warps consecutive segments of 16 (fp32: 8) tokens, each of which
//   1. turns its segment, which cp.async has brought into shared memory two rounds ago, into gates and increments in registers,
//      and asks for the segment two rounds on;
//   2. gets the state that enters the segment;
//   3. walks the segment from that state and writes the outputs.
// Where there are sequences enough for the device, a CTA has one to itself and step 2 is a box that the warp in front fills when it
// has walked its segment (Mail): no warp waits for another but for that.  Forward / backward of B=8, T=4096, C=2048, bf16, sigmoid: 72 / 118 us,
// 0.94 / 0.92 of the measured copy rate (ncu's clock; between events around a call whose operands are not in L2, as the figures further
// down, 80 / 131); 256 CTAs on 296 places.  A segment's way through the chain takes 333 cycles (265 backward), which
// is what bounds a long sequence then: 11 ns a token.
// Where there are fewer, a cluster of up to eight CTAs shares a sequence, tile by tile.  The recurrence is associative: a stretch of
// tokens acts on the state entering it as h -> A h + b.  The warps reduce their segments to (A, b), the last one sends the whole tile's to
// every CTA of the cluster (st.async onto an mbarrier there), and everyone carries the state over all tiles of the round: one hop,
// whatever the size of the cluster.  One sequence of 32768 tokens, C=2048: 96 us in 32 clusters of eight, 0.65 of the copy rate; 48 % of issue slots.
// A round is a chain of steps that wait for one another (gates, summary, barrier, the joins of eight segments, hop, the joins of eight CTAs, walk),
// which two CTAs an SM hide in part; the hop is 8 us of the 96.
// Segments of 16 tokens and a pair of channels a lane are what 128 registers hold; with 8 tokens the work around a segment makes the forward
// 125 us instead of 82, with 16 warps a CTA 107 (both measured in the form with barriers).
//
// Backward: dh_t = gy_t + [t == length-1] gs + c_{t+1},  c_t = start_t ? 0 : a_t dh_t.  The states are recomputed in segments of 8
// tokens from the state entering each, which the forward keeps (4 bytes per 8 tokens and channel: a twelfth of a bf16 forward's traffic, a
// twentieth of the backward's); c runs over the segments from the last to the first as the state does forward.
//
// A start flag cuts by a select, not by a factor of 0: what is no number in front of it ends there.
#include <limits.h>

#include <initializer_list>
#include <type_traits>

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
constexpr int kKept = 8;                   // tokens per kept state, and of a backward segment
constexpr int kMaxCluster = 8;
constexpr int kStages = 2;
constexpr int kWaitRanOut = 3;             // status word: a wait for the warp in front, or for the other CTAs of a cluster

// two channels, as they lie in shared memory
__device__ __forceinline__ F2 pair_at(const float* p) { return *reinterpret_cast<const F2*>(p); }
__device__ __forceinline__ F2 pair_at(const __nv_bfloat16* p) { return unpack_pair(*reinterpret_cast<const uint32_t*>(p)); }
__device__ __forceinline__ void store_pair(float* p, F2 a) { *reinterpret_cast<F2*>(p) = a; }
__device__ __forceinline__ void store_pair(__nv_bfloat16* p, F2 a) {
    const float2 q = parts(a);
    *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(q.x, q.y);
}

constexpr int kSigmoidGate = B200WKV_GATE_SIGMOID;
// The gate a, and what the backward needs of it: `w`, for the sigmoid 1 - a (to full relative precision), for the decay -da/df.
template <typename T, int kGate> __device__ __forceinline__ void gate_of(F2 f, F2& a, F2& w) {
    if (kGate == kSigmoidGate) {
        sigmoid_pair<T>(f, a, w);
    } else {
        // (accurate in 16 bits too: the state sums 1 / (1 - a) tokens, and an error of a is that much larger in it)
        const float2 z = parts(f);
        const float e0 = expf(z.x), e1 = expf(z.y), a0 = expf(-e0), a1 = expf(-e1);
        a = make_f2(a0, a1);
        w = make_f2(a0 == 0.f ? 0.f : e0 * a0, a1 == 0.f ? 0.f : e1 * a1);      // (e may be infinite then)
    }
}

struct Stream {                            // rows of C adjacent channels
    const void* p;
    long long batch, token;                // strides in elements
};
struct Problem {
    int B, T, C;
    Stream x, f;
    const float* s0;
    const uint32_t* length;
    const uint8_t* starts;
    int* status;
};

// What a stretch does to the states of two channels: h -> A h + b.  A start flag inside, which drops h, makes both A negative (-0 is).
// Either says it for both: a gate that is no number takes the sign of its channel, whose b is no number then either.
__device__ __forceinline__ bool negative(float A) { return __float_as_uint(A) + 0x80000000u <= 0x7f800000u; }
__device__ __forceinline__ bool cuts(F2 A) {
    const float2 q = parts(A);
    return negative(q.x) || negative(q.y);
}
struct alignas(16) Stretch {
    F2 A, b;
    __device__ __forceinline__ static Stretch nothing() { return {both(1.f), both(0.f)}; }
    __device__ __forceinline__ F2 of_uncut(F2 h) const { return fma2(A, h, b); }
    __device__ __forceinline__ F2 of(F2 h) const { return cuts(A) ? b : fma2(A, h, b); }
    __device__ __forceinline__ Stretch then(const Stretch& n) const { return {cuts(n.A) ? both(-1.f) : mul2(A, n.A), n.of(b)}; }
};

// A CTA's tiles of one stream on their way to shared memory, each warp its segment: kSeg rows of 64 channels, zeros behind the sequence's
// end and the last channel.  Addresses are a base that is the same for the CTA and 32 bits of the lane's own, where a tile of whole rows is
// that near.  Rows travel as the 16-byte chunks that they lie in.
__device__ __forceinline__ void copy_chunk(uint32_t to, const char* from, int valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(valid) : "memory");
}
// Rows that begin anywhere (kPiece 2 or 4: on what) are a chunk more, and what lies in front of them in it comes along unused (allocations begin
// on 16 bytes, so it is there).  Forward / backward in us, in front of them with copies of 4 bytes and, for rows that begin on 2, of single elements:
// bf16, B=1, T=8191, C=1001 64 / 98 and 47 / 75; B=16, T=1024, C=1001 54 / 86 and 37 / 53; B=4, T=2048, C=2046 48 / 72 and 40 / 61; fp32, B=8,
// T=2048, C=1001 69 / 113 and 57 / 71.  (Words instead of elements for the outputs of such rows too: 51 / 88 -> 57 / 102, not taken.)
template <typename T, int kPiece, int kSeg> struct Feed {
    static constexpr int kChunks = kWide * (int)sizeof(T) / 16, kRow = (kChunks + 1) * 16;      // of a row; bytes in shared memory
    static constexpr int kRows = 32 / kChunks;                          // at a time
    const char* base;                      // the chunk of the CTA's first channel in token 0
    long long stride;                      // bytes from token to token
    uint32_t off;                          // the lane's first row in a tile
    int shift, step;                       // of a row in its first chunk: of token 0, and from token to token
    int bytes;                             // of the channels that there are
    bool near;
    __device__ __forceinline__ static int row() { return (int)(threadIdx.x & 31) / kChunks; }
    __device__ __forceinline__ static int chunk() { return (int)(threadIdx.x & 31) % kChunks; }
    __device__ __forceinline__ Feed(const void* p, long long batch, long long token, int bi, int c0, int C)
        : base((const char*)p + (bi * batch + c0) * (long long)sizeof(T)), stride(token * (long long)sizeof(T)), bytes((C - c0) * (int)sizeof(T)) {
        shift = (int)(uintptr_t)base & 15;
        step = (int)stride & 15;
        base -= shift;
        off = (threadIdx.x / 32 * kSeg + row()) * (uint32_t)stride + shift;
        near = stride * (kSeg * kWarps) < (1LL << 31) && bytes >= kRow;
    }
    // of the warp's i-th row (its segment begins at a multiple of eight tokens)
    __device__ __forceinline__ int shift_of(int i) const { return (shift + i * step) & 15; }
    // chunk k of the warp's i-th row, where not all of it may be there
    __device__ __forceinline__ void edge(uint32_t to, int t0, int i, int k, int Tlen) const {
        const int left = t0 + i < Tlen ? bytes + shift_of(i) - 16 * k : 0, valid = left < 0 ? 0 : left < 16 ? left : 16;
        copy_chunk(to + i * kRow + 16 * k, base + (valid ? (((t0 + i) * stride + shift) & ~15LL) + 16 * k : 0), valid);
    }
    // the tile that begins at t0; `to`: the warp's rows in shared memory
    __device__ __forceinline__ void fetch(uint32_t to, int t0, int Tlen) const {
        const int seg = (int)(threadIdx.x / 32) * kSeg, lane = threadIdx.x & 31;
        if (near && t0 + kSeg * kWarps <= Tlen) {
            const char* const tile = base + t0 * stride;
            const uint32_t down = (uint32_t)(kRows * stride), into = to + row() * kRow + 16 * chunk();
            uint32_t at = off;
#pragma unroll
            for (int i = 0; i < kSeg; i += kRows, at += down) copy_chunk(into + i * kRow, tile + ((at & ~15u) + 16 * chunk()), 16);
            if (lane < kSeg) copy_chunk(to + lane * kRow + 16 * kChunks, tile + ((((seg + lane) * (uint32_t)stride + shift) & ~15u) + 16 * kChunks), 16);
        } else {
            for (int i = 0; i < kSeg; i += kRows) edge(to, t0 + seg, i + row(), chunk(), Tlen);
            if (lane < kSeg) edge(to, t0 + seg, lane, kChunks, Tlen);
        }
    }
    // the lane's two channels of the warp's i-th row; `rows`: where they would be in the first one if it began on 16 bytes
    __device__ __forceinline__ F2 at(const unsigned char* rows, int i) const {
        const unsigned char* const q = rows + i * kRow + shift_of(i);
        if constexpr (sizeof(T) == 4) {
            return make_f2(((const float*)q)[0], ((const float*)q)[1]);
        } else if constexpr (kPiece == 4) {
            return pair_at((const __nv_bfloat16*)q);
        } else {                           // a word, or the halves of two
            const uint32_t half = (uint32_t)(uintptr_t)q & 2;
            const uint32_t* const word = (const uint32_t*)(q - half);
            return unpack_pair(__funnelshift_r(word[0], word[1], half * 8));
        }
    }
};
// Rows that begin on 16 bytes.
template <typename T, int kSeg> struct Feed<T, 16, kSeg> {
    static constexpr int kPer = 16 / (int)sizeof(T), kChunks = kWide / kPer, kRow = kChunks * 16, kRows = 32 / kChunks;
    const char* base;                      // token 0 of the CTA's channels
    long long stride;
    uint32_t off;                          // the lane's first chunk in a tile
    int left;                              // channels that there are
    bool near;
    __device__ __forceinline__ static int row() { return (int)(threadIdx.x & 31) / kChunks; }
    __device__ __forceinline__ static int channel() { return (int)(threadIdx.x & 31) % kChunks * kPer; }
    __device__ __forceinline__ Feed(const void* p, long long batch, long long token, int bi, int c0, int C)
        : base((const char*)p + (bi * batch + c0) * (long long)sizeof(T)), stride(token * (long long)sizeof(T)), left(C - c0) {
        near = stride * (kSeg * kWarps) < (1LL << 31) && left >= kWide;
        off = (uint32_t)((threadIdx.x / 32 * kSeg + row()) * (uint32_t)stride + channel() * sizeof(T));
    }
    __device__ __forceinline__ void fetch(uint32_t to, int t0, int Tlen) const {
        to += row() * kRow + channel() * (int)sizeof(T);
        if (near && t0 + kSeg * kWarps <= Tlen) {
            const char* const tile = base + t0 * stride;
            const uint32_t down = (uint32_t)(kRows * stride);
            uint32_t at = off;
#pragma unroll
            for (int i = 0; i < kSeg; i += kRows, at += down) copy_chunk(to + i * kRow, tile + at, 16);
        } else {
            const int first = t0 + (int)(threadIdx.x / 32) * kSeg + row();
            for (int i = 0; i < kSeg; i += kRows) {
                const bool valid = first + i < Tlen && channel() < left;
                copy_chunk(to + i * kRow, base + (valid ? (first + i) * stride + channel() * (long long)sizeof(T) : 0), valid ? 16 : 0);
            }
        }
    }
    __device__ __forceinline__ F2 at(const unsigned char* rows, int i) const { return pair_at((const T*)rows + i * kWide); }
};
__device__ __forceinline__ void fetched() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void wait_fetched() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
    __syncwarp();
}

// A pair of channels of a dense row; single elements where pairs do not fit the row (kPiece one element), whose last may have no second.
// (A lane behind the last channel goes along with the last pair, and writes what that writes.)
template <typename T, int kPiece> __device__ __forceinline__ void put(T* p, F2 a, int channels) {
    if constexpr (kPiece >= 2 * (int)sizeof(T)) {
        store_pair(p, a);
    } else {
        const float2 q = parts(a);
        p[0] = from_f32<T>(q.x);
        if (channels > 1) p[1] = from_f32<T>(q.y);
    }
}
// kPair: both at once, where C is even and the array begins on 8 bytes
template <bool kPair = false> __device__ __forceinline__ F2 get_state(const float* p, int channels) {
    if (kPair) return *reinterpret_cast<const F2*>(p);
    return make_f2(p != nullptr ? p[0] : 0.f, p != nullptr && channels > 1 ? p[1] : 0.f);
}
template <bool kPair = false> __device__ __forceinline__ void put_state(float* p, F2 h, int channels) {
    if (kPair) {
        *reinterpret_cast<F2*>(p) = h;
    } else {
        const float2 q = parts(h);
        p[0] = q.x;
        if (channels > 1) p[1] = q.y;
    }
}

// Whether the lane's token of a segment has a start flag; read well before the segment's mask (bit i = token t0 + i) is made of it.
template <int kSeg> __device__ __forceinline__ bool start_flag(const uint8_t* ns, int t0, int T) {
    const int lane = threadIdx.x & 31;
    return ns != nullptr && lane < kSeg && t0 + lane < T && ns[t0 + lane] != 0;
}

// What the CTAs of a cluster tell one another: the stretches of a round's tiles.  Two rounds' worth: a CTA sends a round's only when
// it has those of the round in front from everyone, who by then have used the round before that.
struct Exchange {
    Stretch tiles[2][kMaxCluster][32];
    uint64_t bar[2];
    __device__ __forceinline__ void open() {
        if (threadIdx.x == 0) {
            mbar_init(&bar[0], 1);
            mbar_init(&bar[1], 1);
            mbar_init_fence();
        }
        cluster_sync();
    }
    __device__ __forceinline__ void send(int round, int rank, int ranks, const Stretch& tile, int lane) {   // by one warp
        uint64_t* const mine = &bar[round & 1];
        if (lane == 0) mbar_expect_tx(mine, (uint32_t)ranks * 32 * sizeof(Stretch));
        const float2 A = parts(tile.A), b = parts(tile.b);
        for (int q = 0; q < ranks; ++q) store_in_cta(in_cta(&tiles[round & 1][rank][lane], q), make_float4(A.x, A.y, b.x, b.y), in_cta(mine, q));
    }
    __device__ __forceinline__ void wait(int round, bool& lost, int* status) {
        if (lost || mbar_wait_cluster(&bar[round & 1], (round >> 1) & 1)) return;
        lost = true;
        if (status != nullptr) *status = kWaitRanOut;
    }
    // no CTA leaves while others may still send to it
    __device__ __forceinline__ void close() { cluster_sync(); }
};

// Grid: x the 64 channels and, inside, the CTAs of a cluster; y and z the sequence
struct Place {
    int rank, ranks, lane, warp, bi, c0, col, channels, L;
    __device__ __forceinline__ Place(const Problem& p) {
        rank = (int)cluster_rank(); ranks = (int)cluster_size();
        lane = threadIdx.x & 31;
        warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
        bi = blockIdx.y + blockIdx.z * gridDim.y;
        unsigned slab;
        asm("mov.u32 %0, %%clusterid.x;" : "=r"(slab));
        c0 = (int)slab * kWide;
        col = min(2 * lane, (p.C - c0 - 1) & ~1);
        channels = p.C - c0 - col;
        L = p.length != nullptr && bi < p.B ? (int)min(p.length[bi], (uint32_t)p.T) : p.T;
    }
    __device__ __forceinline__ size_t state(const Problem& p) const { return (size_t)bi * p.C + c0 + col; }      // in a dense (B, C) array
};
struct Plain { static constexpr bool value = true; };      // a whole segment without a start flag in which the returned state is not taken
struct Marked { static constexpr bool value = false; };

// The segments of a tile by what they do to a state, in the order in which it meets them.
struct Chain {
    Stretch s[kWarps][32];
    __device__ __forceinline__ Stretch& of(int place) { return s[place][threadIdx.x & 31]; }
    // what the first `n` segments do together; `marked`: a start flag is among the tile's
    __device__ __forceinline__ Stretch first(int n, bool marked) const {
        Stretch t = Stretch::nothing();
        if (!marked) {
#pragma unroll
            for (int j = 0; j < kWarps; ++j)
                if (j < n) {
                    const Stretch next = s[j][threadIdx.x & 31];
                    t = {mul2(t.A, next.A), next.of_uncut(t.b)};
                }
        } else {
            for (int j = 0; j < n; ++j) t = t.then(s[j][threadIdx.x & 31]);
        }
        return t;
    }
};

// How the state goes from warp to warp where one CTA has the sequence: in turn, each with its segment.  A warp's box is written again
// when its last content has gone around through all of them.
struct Mail {
    F2 box[kWarps][32];
    uint64_t bar[kWarps];
    __device__ __forceinline__ void open() {
        if (threadIdx.x == 0)
            for (int w = 0; w < kWarps; ++w) mbar_init(&bar[w], 1);
        __syncthreads();
    }
    __device__ __forceinline__ F2 take(int warp, int phase, bool& lost, int* status) {
        if (!lost && !mbar_wait(&bar[warp], phase & 1)) {
            lost = true;
            if (status != nullptr) *status = kWaitRanOut;
        }
        return box[warp][threadIdx.x & 31];
    }
    __device__ __forceinline__ void pass(int to, F2 h) {
        box[to][threadIdx.x & 31] = h;
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(&bar[to]);
    }
};

template <typename T> constexpr int kFwdSeg = sizeof(T) == 2 ? 16 : 8;
constexpr int kBwdSeg = kKept;

// kTurn: one CTA has the sequence, and its warps take the state over from one another, so that nothing is summarised and no barrier
// joins them.  Else a cluster shares it.
template <typename T, int kGate, int kPiece, bool kTurn>
__global__ void __launch_bounds__(kWarps * 32, 2)
gated_fwd_kernel(const Problem p, T* __restrict__ y, float* __restrict__ s_out, float* __restrict__ kept) {
    constexpr int kSeg = kFwdSeg<T>, kTile = kSeg * kWarps, kRow = Feed<T, kPiece, kSeg>::kRow, kRoom = 2 * kSeg * kRow;
    extern __shared__ __align__(128) unsigned char dynamic[];
    __shared__ std::conditional_t<kTurn, Mail, Exchange> ex;
    __shared__ std::conditional_t<kTurn, char, Chain> chain[2];
    const Place at(p);
    if (at.bi >= p.B) return;              // (a whole cluster)
    const int lane = at.lane, warp = at.warp, rank = kTurn ? 0 : at.rank, ranks = kTurn ? 1 : at.ranks, c0 = at.c0;
    const size_t state = at.state(p);
    const int tiles = (p.T + kTile - 1) / kTile, rounds = (tiles + ranks - 1) / ranks;
    const Feed<T, kPiece, kSeg> fx(p.x.p, p.x.batch, p.x.token, at.bi, c0, p.C), ff(p.f.p, p.f.batch, p.f.token, at.bi, c0, p.C);
    unsigned char* const room = dynamic + warp * kStages * kRoom;
    const auto ask = [&](int round) {
        if (round < rounds) {
            const uint32_t to = smem_u32(room) + round % kStages * kRoom;
            fx.fetch(to, (round * ranks + rank) * kTile, p.T);
            ff.fetch(to + kSeg * kRow, (round * ranks + rank) * kTile, p.T);
        }
        fetched();
    };
    for (int i = 0; i < kStages; ++i) ask(i);
    F2 carry = get_state(p.s0 != nullptr ? p.s0 + state : nullptr, at.channels);      // state entering the round (kTurn: the sequence)
    if (at.L == 0 && warp == 0 && rank == 0) put_state(s_out + state, carry, at.channels);
    ex.open();
    bool lost = false;
    const uint8_t* const ns = p.starts != nullptr ? p.starts + (size_t)at.bi * p.T : nullptr;
    const uint32_t down = p.C * (uint32_t)sizeof(T), own_off = warp * kSeg * down + at.col * (uint32_t)sizeof(T);
    const int states = (p.T + kKept - 1) / kKept;
    for (int round = 0; round < rounds; ++round) {
        const int tile = (round * ranks + rank) * kTile, t0 = tile + warp * kSeg, n = max(0, min(kSeg, p.T - t0));
        const bool flag = start_flag<kSeg>(ns, t0, p.T);
        // 1. gates and increments
        F2 a[kSeg], u[kSeg];
        wait_fetched<kStages - 1>();
        const unsigned char* const from = room + round % kStages * kRoom + at.col * (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < kSeg; ++i) {
            const F2 x = fx.at(from, i);
            F2 w;
            gate_of<T, kGate>(ff.at(from + kSeg * kRow, i), a[i], w);
            u[i] = kGate == kSigmoidGate ? mul2(w, x) : x;
        }
        __syncwarp();                      // the segment has been read
        ask(round + kStages);
        const uint32_t starts = __ballot_sync(0xffffffffu, flag);
        const bool plain = n == kSeg && starts == 0 && (at.L <= t0 || at.L > t0 + kSeg);
        // 2. the state that enters the segment
        F2 h;
        if constexpr (kTurn) {
            h = warp == 0 && round == 0 ? carry : ex.take(warp, warp == 0 ? round - 1 : round, lost, p.status);
        } else {
            const int parity = round & 1;
            F2 A = both(1.f), b = both(0.f);
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
            chain[parity].of(warp) = Stretch{A, b};
            const bool marked = __syncthreads_or(starts != 0);   // a start flag in the tile
            if (warp == kWarps - 1) ex.send(round, rank, ranks, chain[parity].first(kWarps, marked), lane);
            const Stretch front = chain[parity].first(warp, marked);
            ex.wait(round, lost, p.status);
#pragma unroll
            for (int q = 0; q < kMaxCluster; ++q) {
                if (q >= ranks) break;
                if (q == rank) h = carry;
                carry = ex.tiles[parity][q][lane].of(carry);
            }
            h = front.of(h);
        }
        // 3. the states; outputs, and the states that are kept
        char* const to = (char*)y + (((long long)at.bi * p.T + tile) * p.C + c0) * (long long)sizeof(T);
        const F2 first = h;
        const auto walk = [&](auto kind) {
#pragma unroll
            for (int i = 0; i < kSeg; ++i) {
                const bool start = !kind.value && ((starts >> i) & 1u);
                if (kind.value || i < n) u[i] = h = start ? u[i] : fma2(a[i], h, u[i]);
            }
            if constexpr (kTurn) ex.pass((warp + 1) % kWarps, h);
            uint32_t off = own_off;
#pragma unroll
            for (int i = 0; i < kSeg; ++i, off += down) {
                if (kind.value || i < n) {
                    put<T, kPiece>((T*)(to + off), u[i], at.channels);
                    if (kept != nullptr && i % kKept == 0)
                        put_state<(kPiece > 4)>(kept + ((long long)at.bi * states + t0 / kKept + i / kKept) * p.C + c0 + at.col, i == 0 ? first : u[i == 0 ? 0 : i - 1], at.channels);
                }
                if (!kind.value && t0 + i == at.L - 1) put_state(s_out + state, u[i], at.channels);
            }
        };
        if (plain) walk(Plain()); else walk(Marked());
    }
    if constexpr (!kTurn) ex.close();
}

template <typename T, int kGate, int kPiece, bool kTurn>
__global__ void __launch_bounds__(kWarps * 32, 2)
gated_bwd_kernel(const Problem p, const T* __restrict__ gy, const float* __restrict__ gs, const float* __restrict__ kept,
                 T* __restrict__ dx, T* __restrict__ df, float* __restrict__ ds0) {
    constexpr int kSeg = kBwdSeg, kTile = kSeg * kWarps, kRow = Feed<T, kPiece, kSeg>::kRow, kRoom = 3 * kSeg * kRow;
    extern __shared__ __align__(128) unsigned char dynamic[];
    __shared__ std::conditional_t<kTurn, Mail, Exchange> ex;
    __shared__ std::conditional_t<kTurn, char, Chain> back[2];
    const Place at(p);
    if (at.bi >= p.B) return;              // (a whole cluster)
    const int lane = at.lane, warp = at.warp, rank = kTurn ? 0 : at.rank, ranks = kTurn ? 1 : at.ranks, c0 = at.c0;
    const size_t state = at.state(p);
    const int tiles = (p.T + kTile - 1) / kTile, rounds = (tiles + ranks - 1) / ranks, states = (p.T + kKept - 1) / kKept;
    const Feed<T, kPiece, kSeg> fx(p.x.p, p.x.batch, p.x.token, at.bi, c0, p.C), ff(p.f.p, p.f.batch, p.f.token, at.bi, c0, p.C);
    const Feed<T, kPiece, kSeg> fg(gy, (long long)p.T * p.C, p.C, at.bi, c0, p.C);
    unsigned char* const room = dynamic + warp * kStages * kRoom;
    // rounds are taken from the last to the first; `done` of them lie behind
    const auto ask = [&](int done) {
        if (done < rounds) {
            const uint32_t to = smem_u32(room) + done % kStages * kRoom;
            const int tile = ((rounds - 1 - done) * ranks + rank) * kTile;
            fx.fetch(to, tile, p.T);
            ff.fetch(to + kSeg * kRow, tile, p.T);
            if (gy != nullptr) fg.fetch(to + 2 * kSeg * kRow, tile, p.T);
        }
        fetched();
    };
    const auto entering = [&](int done) {  // the kept state in front of the warp's segment
        const int seg = ((rounds - 1 - done) * ranks + rank) * kWarps + warp;
        return done < rounds && seg < states ? get_state<(kPiece > 4)>(kept + ((long long)at.bi * states + seg) * p.C + c0 + at.col, at.channels) : both(0.f);
    };
    if (gy == nullptr)                     // nothing is fetched there, and zeros are read
        for (int i = 0; i < kStages; ++i)
            for (int j = lane; j < kSeg * kRow / 4; j += 32) ((uint32_t*)(room + i * kRoom + 2 * kSeg * kRow))[j] = 0;
    for (int i = 0; i < kStages; ++i) ask(i);
    F2 next = entering(0), carry = both(0.f);                    // carry: c entering the round from behind
    const F2 gstate = get_state(gs != nullptr ? gs + state : nullptr, at.channels);
    ex.open();
    bool lost = false;
    const uint8_t* const ns = p.starts != nullptr ? p.starts + (size_t)at.bi * p.T : nullptr;
    const uint32_t down = p.C * (uint32_t)sizeof(T), own_off = warp * kSeg * down + at.col * (uint32_t)sizeof(T);
    for (int done = 0; done < rounds; ++done) {
        const int tile = ((rounds - 1 - done) * ranks + rank) * kTile, t0 = tile + warp * kSeg, n = max(0, min(kSeg, p.T - t0));
        // (asked for behind the gates, as the forward does, the mask costs the registers that the gates are short of: 129 -> 148 us)
        const uint32_t starts = __ballot_sync(0xffffffffu, start_flag<kSeg>(ns, t0, p.T));
        const bool plain = n == kSeg && starts == 0 && (at.L <= t0 || at.L > t0 + kSeg);
        F2 h = next;
        next = entering(done + 1);
        // 1. gates, states, and in the place of x what df is dx times of
        F2 a[kSeg], w[kSeg], x[kSeg], g[kSeg];
        wait_fetched<kStages - 1>();
        const unsigned char* const from = room + done % kStages * kRoom + at.col * (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < kSeg; ++i) {
            x[i] = fx.at(from, i);
            gate_of<T, kGate>(ff.at(from + kSeg * kRow, i), a[i], w[i]);
            g[i] = fg.at(from + 2 * kSeg * kRow, i);
        }
        __syncwarp();                      // the segment has been read
        ask(done + kStages);
        const auto replay = [&](auto kind) {
#pragma unroll
            for (int i = 0; i < kSeg; ++i) {
                if (!kind.value) {
                    if (i >= n) { a[i] = both(1.f); w[i] = x[i] = both(0.f); }
                    if (t0 + i == at.L - 1) g[i] = add2(g[i], gstate);
                }
                const bool start = !kind.value && ((starts >> i) & 1u);
                const F2 in = start ? both(0.f) : h, u = kGate == kSigmoidGate ? mul2(w[i], x[i]) : x[i];
                h = start ? u : fma2(a[i], h, u);
                if (kGate == kSigmoidGate) x[i] = mul2(fma2(x[i], both(-1.f), in), a[i]);
                else x[i] = start ? both(0.f) : mul2(mul2(in, w[i]), both(-1.f));
            }
        };
        if (plain) replay(Plain()); else replay(Marked());
        // 2. what comes to the segment from behind
        F2 e;
        if constexpr (kTurn) {
            e = done == 0 && warp == kWarps - 1 ? carry : ex.take(warp, warp == kWarps - 1 ? done - 1 : done, lost, p.status);
        } else {
            const int parity = done & 1;
            F2 A = both(1.f), c = both(0.f);
            const auto summarise = [&](auto kind) {
#pragma unroll
                for (int i = kSeg - 1; i >= 0; --i) {
                    const bool start = !kind.value && ((starts >> i) & 1u);
                    A = start ? both(-1.f) : mul2(A, a[i]);
                    c = start ? both(0.f) : mul2(a[i], add2(g[i], c));
                }
            };
            if (plain) summarise(Plain()); else summarise(Marked());
            back[parity].of(kWarps - 1 - warp) = Stretch{A, c};
            const bool marked = __syncthreads_or(starts != 0);   // a start flag in the tile
            if (warp == 0) ex.send(done, rank, ranks, back[parity].first(kWarps, marked), lane);
            const Stretch rear = back[parity].first(kWarps - 1 - warp, marked);
            ex.wait(done, lost, p.status);
#pragma unroll
            for (int q = kMaxCluster - 1; q >= 0; --q) {
                if (q >= ranks) continue;
                if (q == rank) e = carry;
                carry = ex.tiles[parity][q][lane].of(carry);
            }
            e = rear.of(e);
        }
        // 3. back through the segment
        const long long tile_at = (((long long)at.bi * p.T + tile) * p.C + c0) * (long long)sizeof(T);
        char *const to_x = (char*)dx + tile_at, *const to_f = (char*)df + tile_at;
        const auto walk = [&](auto kind) {
#pragma unroll
            for (int i = kSeg - 1; i >= 0; --i) {
                g[i] = add2(g[i], e);
                e = !kind.value && ((starts >> i) & 1u) ? both(0.f) : mul2(a[i], g[i]);
            }
            if constexpr (kTurn) ex.pass((warp + kWarps - 1) % kWarps, e);
            uint32_t off = own_off;
#pragma unroll
            for (int i = 0; i < kSeg; ++i, off += down) {
                const F2 o = kGate == kSigmoidGate ? mul2(g[i], w[i]) : g[i], of = mul2(o, x[i]);
                if (kind.value || i < n) {
                    put<T, kPiece>((T*)(to_x + off), o, at.channels);
                    put<T, kPiece>((T*)(to_f + off), of, at.channels);
                }
            }
        };
        if (plain) walk(Plain()); else walk(Marked());
        if (t0 == 0) put_state(ds0 + state, at.L == 0 ? add2(e, gstate) : e, at.channels);
    }
    if constexpr (!kTurn) ex.close();
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
        const F2 x2 = make_f2(to_f32(rx.q[v]), to_f32(rx.q[v1])), s2 = make_f2(rs.q[v], rs.q[v1]);
        F2 a, w;
        gate_of<T, kGate>(make_f2(to_f32(rf.q[v]), to_f32(rf.q[v1])), a, w);
        const F2 u = kGate == kSigmoidGate ? mul2(w, x2) : x2;
        const float2 out = parts(start ? u : fma2(a, s2, u));
        ry.q[v] = from_f32<T>(out.x);
        ry.q[v1] = from_f32<T>(out.y);
        rh.q[v] = keep ? rs.q[v] : out.x;
        rh.q[v1] = keep ? rs.q[v1] : out.y;
    }
    *(Few<T, V>*)(y + (size_t)bi * C + c) = ry;
    *(Few<float, V>*)(s_out + bi * s_out_stride + c) = rh;
}

// How many clusters of n CTAs a kernel has on the device at a time, asked once per device and kernel (which sets its shared memory too).
struct Residency {
    DeviceOnce once;
    int clusters[kMaxDevices][kMaxCluster + 1];
    template <typename Kernel> const int* of(Kernel kern, size_t smem, int largest) {
        const int dev = current_device();
        if (dev < 0) return nullptr;
        const bool ok = once.ok([&]() {
            const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
            for (int n = 1; n <= largest; ++n) {
                cudaLaunchAttribute attr[1];
                cudaLaunchConfig_t cfg = config(attr, n, dim3(n), smem, nullptr);
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
    static cudaLaunchConfig_t config(cudaLaunchAttribute* attr, int ranks, dim3 grid, size_t smem, cudaStream_t st) {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = ranks; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = grid;
        cfg.blockDim = dim3(kWarps * 32);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        return cfg;
    }
};
// CTAs of a cluster: those with which the last sequence is done soonest, by the rounds that it takes (and one to begin with) and the waves of
// clusters in front of it; the smaller of equals.  One CTA alone takes half of a cluster's time for a round.  Forward / backward in us with one CTA a
// sequence and with clusters, bf16: B=4, T=1024, C=2048 20 / 29 and 25 / 31 (of two); B=16, T=512, C=768 16 / 22 and 27 / 33 (two); B=2, T=8192,
// C=1024 98 / 156 and 35 / 51 (eight); B=1, T=2000, C=2560 30 and 21 (six); B=8, T=1024, C=1001 25 / 37 and 30 / 41 (two); fp32, B=4, T=2048, C=2048
// 43 / 64 and 45 / 80 (two); B=8, T=2048, C=1001 49 / 73 and 55 / 107 (two); the rule's miss: B=3, T=1023, C=1001 backward 37 and 33 (two; all of these
// with the sigmoid gate, the decay gate takes up to 10 % more).
// units: 64 channels of a sequence each; tiles: of one of them.
int ranks_of(const int* alone, const int* resident, long long units, int tiles) {
    constexpr double kAlone = 0.5;
    int best = 1;
    double least = (double)((units + alone[1] - 1) / alone[1]) * (kAlone * tiles + 1);
    for (int n = 2; n <= kMaxCluster && n <= tiles; ++n) {
        if (resident[n] < 1) continue;
        const double rounds = (double)((units + resident[n] - 1) / resident[n]) * ((tiles + n - 1) / n + 1);
        if (rounds < least) { least = rounds; best = n; }
    }
    return best;
}
// A direction's two kernels, and how many of them the device takes.
template <bool kForward, typename T, int kGate, int kPiece> struct Forms {
    static constexpr int kSeg = kForward ? kFwdSeg<T> : kBwdSeg, kTile = kSeg * kWarps;
    static constexpr size_t kSmem = (size_t)kStages * (kForward ? 2 : 3) * kTile * Feed<T, kPiece, kSeg>::kRow;
    template <bool kTurn> static constexpr auto kernel() {
        if constexpr (kForward) return &gated_fwd_kernel<T, kGate, kPiece, kTurn>;
        else return &gated_bwd_kernel<T, kGate, kPiece, kTurn>;
    }
    static bool resident(const int*& alone, const int*& clusters) {
        static Residency residency[2];
        alone = residency[0].of(kernel<true>(), kSmem, 1);
        clusters = residency[1].of(kernel<false>(), kSmem, kMaxCluster);
        return alone != nullptr && clusters != nullptr && alone[1] >= 1;
    }
};
template <bool kForward, typename T, int kGate, int kPiece, typename... Args> int launch(cudaStream_t st, const Problem& p, Args... args) {
    typedef Forms<kForward, T, kGate, kPiece> F;
    const int *alone, *clusters;
    if (!F::resident(alone, clusters)) return B200WKV_ELAUNCH;
    // (the choice goes by the length of the rows, so that results do not depend on where operands lie)
    if (kPiece < 16 && p.C * sizeof(T) % 16 == 0 && !Forms<kForward, T, kGate, 16>::resident(alone, clusters)) return B200WKV_ELAUNCH;
    const int slabs = (p.C + kWide - 1) / kWide, ranks = ranks_of(alone, clusters, (long long)p.B * slabs, (p.T + F::kTile - 1) / F::kTile);
    const unsigned y = p.B < 65535 ? p.B : 65535;
    cudaLaunchAttribute attr[1];
    const cudaLaunchConfig_t cfg = Residency::config(attr, ranks, dim3((unsigned)slabs * ranks, y, (p.B + y - 1) / y), F::kSmem, st);
    return cudaLaunchKernelEx(&cfg, ranks > 1 ? F::template kernel<false>() : F::template kernel<true>(), p, args...) == cudaSuccess ? B200WKV_OK : B200WKV_ELAUNCH;
}
// The widest pieces that every row of these begins on.
int piece_of(int C, int element, std::initializer_list<const void*> streams, std::initializer_list<long long> strides) {
    uintptr_t bits = (uintptr_t)C * element;
    for (const void* q : streams) bits |= reinterpret_cast<uintptr_t>(q);
    for (long long s : strides) bits |= (uintptr_t)s * element;
    return bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 2;
}

template <typename T, int kGate, int kPiece> int fwd(cudaStream_t st, const Problem& p, void* y, float* s_out, float* kept) {
    return launch<true, T, kGate, kPiece>(st, p, (T*)y, s_out, kept);
}
template <typename T, int kGate, int kPiece>
int bwd(cudaStream_t st, const Problem& p, const void* gy, const float* gs, const float* kept, void* dx, void* df, float* ds0) {
    return launch<false, T, kGate, kPiece>(st, p, (const T*)gy, gs, kept, (T*)dx, (T*)df, ds0);
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
    const Problem p = {B, T, C, {x, x_batch, x_token}, {f, f_batch, f_token}, s0, length, ns, wkv7_chunk_status_word()};
    const int piece = piece_of(C, dtype == B200WKV_F32 ? 4 : 2, {x, f, y}, {x_batch, x_token, f_batch, f_token});
    return dtype == B200WKV_F32 ? B200WKV_GATED_PIECE(fwd, float, piece, st, p, y, s_out, (float*)residual)
                                : B200WKV_GATED_PIECE(fwd, __nv_bfloat16, piece, st, p, y, s_out, (float*)residual);
}
int gated_bwd(cudaStream_t st, int dtype, int gate, int B, int T, int C, const void* x, long long x_batch, long long x_token, const void* f,
              long long f_batch, long long f_token, const uint32_t* length, const uint8_t* ns, const void* gy, const float* gs,
              const void* residual, void* dx, void* df, float* ds0) {
    const Problem p = {B, T, C, {x, x_batch, x_token}, {f, f_batch, f_token}, nullptr, length, ns, wkv7_chunk_status_word()};
    const int piece = piece_of(C, dtype == B200WKV_F32 ? 4 : 2, {x, f, gy, dx, df}, {x_batch, x_token, f_batch, f_token});
    return dtype == B200WKV_F32 ? B200WKV_GATED_PIECE(bwd, float, piece, st, p, gy, gs, (const float*)residual, dx, df, ds0)
                                : B200WKV_GATED_PIECE(bwd, __nv_bfloat16, piece, st, p, gy, gs, (const float*)residual, dx, df, ds0);
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
