// The diagonal recurrence over whole sequences, forwards and backwards
// (include/cgdr_recurrence.h).
//
// One cluster of CTAs walks along the tokens of one slab of 32 V channels, a
// segment at a time; a lane owns V channels, a warp 16 consecutive tokens of
// the segment, a CTA of W warps 16 W.  Per segment:
//   1. every warp runs its 16 steps from a zero state and keeps the factor
//      A = prod exp(g) and the end state B, so that the true end state is
//      A h_in + B;
//   2. the CTA's warps join their (A, B) through shared memory, the CTAs
//      theirs through distributed shared memory (every CTA tells all), and
//      everyone folds the state that enters the next segment;
//   3. every warp repeats its 16 steps from its true h_in and stores them.
// x and g are read once and out is written once.  A warp brings its own 16
// rows of the next segments into its own shared memory, by TMA where rows
// allow it (16-byte multiples) and by cp.async otherwise, so the ring needs no
// barrier between warps and the copies run on while the CTA joins.  Every sum
// is taken in a fixed order, so the results are the same on every run.
//
// Pace.  CTAs of neighbouring slabs read and write neighbouring 128 bytes of
// the same rows; once they drift apart, each access opens a DRAM page of its
// own.  So the CTAs of up to four slabs form one hardware cluster, and none is
// more than a segment ahead of its neighbours (a barrier without memory order,
// waited for a segment later): 166 -> 136 us forwards and 303 -> 229 us
// backwards on 4 x 8192 x 4096.  Only where all CTAs are resident at once: with
// several waves it cost 10 % (16 x 1024 x 8192).
//
// Backwards, the same with u_t = exp(g_{t+1}) dh_{t+1} folded from the right
// (the factors A are the same), and with h_{t-1} recomputed from the state
// that the forward pass saved before each 128 tokens.
//
// Sequences.  At a sequence's first token the running state is replaced by
// its initial state, at its last token (backwards) u by d_final_state; a warp
// that does so marks its B as independent of what enters (`cut`), rather than
// relying on A = 0, so that NaN and infinities stay in their sequence.
//
// What bounds it.  On 4 x 8192 x 4096 bf16 DRAM: 135 us forwards, 229 us
// backwards, 5.9 TB/s both.  With fewer slabs than SMs the segments' latency:
// 300 and 500 us on 65536 x 4096 (5.4 TB/s), and on 32768 x 2048 with fp32
// gates 119 and 197 us (4.5 and 4.8).  A border between sequences holds up the
// cluster whose warp meets it by 2 to 4 us: 16 of them 160 and 255 us.
#pragma once

#include <cuda.h>

#include <cstdint>

#include "ptx.cuh"
#include "vec_io.cuh"

namespace cgdr {

constexpr int kScanSteps = 16;     // tokens of a warp and segment; a CTA of W warps has 16 W
constexpr int kScanChunk = 128;    // CGDR_RECURRENCE_CHUNK: tokens between saved states
// CTAs of a cluster at most; backwards fewer, so that two CTAs' shared memory
// fits an SM
constexpr int kScanForwardCluster = 8, kScanBackwardCluster = 4;

struct ScanParams {
    const void *x, *g, *d_out;
    const float *h0, *d_ht;
    const int64_t* cu;       // nullptr: every batch row is one sequence
    void *out, *dx, *dg;
    float *ht, *d_h0, *chunk;
    int64_t B, T, D, N;
    int64_t x_sb, x_st, g_sb, g_st, o_sb, o_st, do_sb, do_st, dx_sb, dx_st, dg_sb, dg_st;
    int64_t h0_sn, ht_sn, dht_sn, dh0_sn;
    int32_t cluster;  // CTAs that share a slab's tokens
    int32_t pace;     // neighbouring slabs in one hardware cluster (1 with cluster > 1)
};

// The warp's index in a register that the compiler knows to be uniform, so
// that row addresses are formed once a warp.
__device__ __forceinline__ int scan_warp() { return __shfl_sync(~0u, static_cast<int>(threadIdx.x / 32), 0); }

// ---- a lane's V channels -------------------------------------------------------------------
// (The packed fp32x2 instructions were tried here: fewer instructions, the same
// time, as each takes the place of two.)

template <int V>
struct Vec {
    float v[V];
    static __device__ __forceinline__ Vec of(float x)
    {
        Vec r;
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[i] = x;
        return r;
    }
};
template <int V>
__device__ __forceinline__ Vec<V> vec_fma(Vec<V> a, Vec<V> b, Vec<V> c)
{
    Vec<V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = fmaf(a.v[i], b.v[i], c.v[i]);
    return r;
}
template <int V>
__device__ __forceinline__ Vec<V> operator*(Vec<V> a, Vec<V> b)
{
    Vec<V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = a.v[i] * b.v[i];
    return r;
}
template <int V>
__device__ __forceinline__ Vec<V> operator+(Vec<V> a, Vec<V> b)
{
    Vec<V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = a.v[i] + b.v[i];
    return r;
}

template <typename T, int V>
__device__ __forceinline__ Vec<V> vec_of(const Pack<T, V>& p)
{
    Vec<V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = to_f32(p.e[i]);
    return r;
}

// exp(g): by the hardware's exponential (within 2 ulp; the argument's own
// rounding adds |g| half-ulps); results below 2^-126 are 0.
template <int V>
__device__ __forceinline__ Vec<V> vec_exp(Vec<V> g)
{
    Vec<V> r;
#pragma unroll
    for (int i = 0; i < V; ++i)
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r.v[i]) : "f"(g.v[i] * 1.4426950408889634f));
    return r;
}

// ---- sequences ------------------------------------------------------------------------

// What a warp knows of the sequences' borders (cu_seqlens, or 0 and T), as it
// walks along the tokens 16 at a time.  The nearest border ahead is kept, so
// they are searched only where one lies in the 16 tokens or behind them, and
// the first 32 borders stay in a register of each lane.
struct ScanBorders {
    int64_t first, last;  // tokens [first, last) belong to sequences
    int64_t ahead;
    int64_t sequence;
    int64_t kept;         // this lane's border among the first 32
    __device__ __forceinline__ ScanBorders(const ScanParams& p, bool reverse)
        : first(0), last(p.T), ahead(reverse ? INT64_MAX : INT64_MIN), sequence(0), kept(border(p, threadIdx.x % 32))
    {
        if (p.cu) {
            first = p.cu[0];
            const int64_t end = p.cu[p.N];
            last = end < p.T ? end : p.T;
        }
    }
    // border i of cu_seqlens, or of 0, T; past the last one none is near
    static __device__ __forceinline__ int64_t border(const ScanParams& p, int64_t i)
    {
        if (!p.cu) return i == 0 ? 0 : i == 1 ? p.T : INT64_MAX;
        return i <= p.N ? p.cu[i] : INT64_MAX;
    }
    // Bit i: a sequence begins or ends before token t + i, 0 <= i <= 16.  Where
    // there is one, lane i holds the sequence of token t + i afterwards: the
    // last one that begins at or before it.
    template <bool REVERSE>
    __device__ __forceinline__ uint32_t at(const ScanParams& p, int64_t b, int64_t t)
    {
        if (REVERSE ? ahead < t : ahead > t + kScanSteps) return 0;
        const int lane = threadIdx.x % 32;
        uint32_t bits = 0;
        int begun = 0;                // sequences that begin at or before token t + lane
        unsigned near = 0xffffffffu;  // distance of the nearest border past the 17 places
        const int64_t n = p.cu ? p.N : 1;
        for (int64_t i0 = 0; i0 <= n; i0 += 32) {
            const int64_t at = i0 == 0 ? kept : border(p, i0 + lane);
            const int64_t d = at == INT64_MAX ? at : at - t;
            const bool here = d >= 0 && d <= kScanSteps;
            if (here) bits |= 1u << d;
            const int64_t far = REVERSE ? -d : d - kScanSteps;
            if (far > 0 && far < near) near = static_cast<unsigned>(far);
            begun += __popc(__ballot_sync(~0u, d < 0));
            if (__any_sync(~0u, here))
#pragma unroll 1
                for (int j = 0; j <= kScanSteps; ++j) {
                    const int add = __popc(__ballot_sync(~0u, here && d <= j));
                    if (lane == j) begun += add;
                }
        }
        near = __reduce_min_sync(~0u, near);
        ahead = REVERSE ? t - near : t + kScanSteps + near;
        const int64_t s = p.cu ? static_cast<int64_t>(begun) - 1 : b;
        sequence = s < 0 ? 0 : s < p.N ? s : p.N - 1;
        return __reduce_or_sync(~0u, bits);
    }
    __device__ __forceinline__ int64_t of(int l) const { return __shfl_sync(~0u, sequence, l); }
    // Bit i: token t + i belongs to no sequence.
    __device__ __forceinline__ uint32_t dead(int64_t t) const
    {
        constexpr uint32_t all = (1u << kScanSteps) - 1;
        const int64_t from = first - t, to = last - t;
        const uint32_t before = from <= 0 ? 0 : from >= kScanSteps ? all : (1u << from) - 1;
        const uint32_t upto = to <= 0 ? 0 : to >= kScanSteps ? all : (1u << to) - 1;
        return (before | ~upto) & all;
    }
};

// Channels c .. c + V of row n of a [N, D] fp32 tensor (zeros without one).
template <int V>
__device__ __forceinline__ Vec<V> scan_load_state(const float* base, int64_t stride, int64_t n, int64_t c, bool mine)
{
    Vec<V> r = Vec<V>::of(0.0f);
    if (base && mine)
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[i] = base[n * stride + c + i];
    return r;
}

template <int V>
__device__ __forceinline__ void scan_store_state(float* base, int64_t stride, int64_t n, int64_t c, bool mine, Vec<V> v)
{
    if (!base || !mine) return;
#pragma unroll
    for (int i = 0; i < V; ++i) base[n * stride + c + i] = v.v[i];
}

// States of empty sequences pass through (`to` from `from`).
template <int V, int W>
__device__ __forceinline__ void scan_empty_sequences(const ScanParams& p, const float* from, int64_t from_s, float* to,
                                                     int64_t to_s, int64_t c, bool mine)
{
    if (!p.cu || !to) return;
    for (int64_t n = threadIdx.x / 32; n < p.N; n += W) {
        if (p.cu[n + 1] > p.cu[n]) continue;
        scan_store_state<V>(to, to_s, n, c, mine, scan_load_state<V>(from, from_s, n, c, mine));
    }
}

// ---- the ring: each warp's own 16 rows -------------------------------------------------------

// Row `l` behind `row`, rows `step` bytes apart.
__device__ __forceinline__ uint64_t scan_row(uint64_t row, uint32_t step, uint32_t l)
{
    uint64_t r;
    asm("mad.wide.u32 %0, %1, %2, %3;" : "=l"(r) : "r"(step), "r"(l), "l"(row));
    return r;
}

// Rows of 32 V channels of one tensor, and how a warp brings 16 of them in.
template <typename T, int V, bool TMA>
struct ScanRows {
    static constexpr int kLane = sizeof(T) * V;
    static constexpr int kBytes = kLane * 32 * kScanSteps;  // of a warp and stage

    // Rows t .. t + 16 of the slab to `to`.  By TMA: one lane calls, rows past
    // the tensor's end are zero, all bytes count on `full`.  By cp.async: all
    // lanes call, each copies what it will read; rows past `end` stay as they
    // are.  `base`: the slab's first channel at token 0.
    static __device__ __forceinline__ void fetch_tma(const CUtensorMap* map, int slab, int t, int b, uint64_t* full,
                                                     uint8_t* to)
    {
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(to)),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(slab), "r"(t), "r"(b), "r"(smem_u32(full))
            : "memory");
    }
    static __device__ __forceinline__ void fetch(const T* base, int64_t stride, int64_t t, int64_t end, uint8_t* to)
    {
        const int lane = threadIdx.x % 32;
        const uint64_t row = reinterpret_cast<uint64_t>(base + t * stride) + lane * kLane;
        const uint32_t step = static_cast<uint32_t>(stride) * sizeof(T);  // below 2^27: checked by the host
        const int count = end - t >= kScanSteps ? kScanSteps : end > t ? static_cast<int>(end - t) : 0;
        to += lane * kLane;
        if constexpr (kLane >= 4) {
            const uint32_t at = smem_u32(to);
            if (count == kScanSteps) {
#pragma unroll
                for (int l = 0; l < kScanSteps; ++l) copy(at + l * 32 * kLane, scan_row(row, step, l));
            } else {
                for (int l = 0; l < count; ++l) copy(at + l * 32 * kLane, scan_row(row, step, l));
            }
        } else {  // two bytes: too small for cp.async
            T e[kScanSteps];
#pragma unroll
            for (int l = 0; l < kScanSteps; ++l)
                if (l < count) e[l] = *reinterpret_cast<const T*>(scan_row(row, step, l));
#pragma unroll
            for (int l = 0; l < kScanSteps; ++l)
                if (l < count) *reinterpret_cast<T*>(to + l * 32 * kLane) = e[l];
        }
    }
    static __device__ __forceinline__ void copy(uint32_t to, uint64_t from)
    {
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(kLane) : "memory");
    }
    static __device__ __forceinline__ Pack<T, V> get(const uint8_t* stage, int l)
    {
        return load_pack<T, V, true>(reinterpret_cast<const T*>(stage + (l * 32 + threadIdx.x % 32) * kLane));
    }
};

__device__ __forceinline__ void scan_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

template <int PENDING>
__device__ __forceinline__ void scan_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

// A CTA's step: waits until the cluster's CTAs have begun the segment before.
__device__ __forceinline__ void scan_pace(const ScanParams& p, bool first)
{
    if (p.pace == 1) return;
    if (!first) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void scan_pace_end(const ScanParams& p)
{
    if (p.pace > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

constexpr uint64_t kScanWaitNs = 2000000000ull;

// Waits for a barrier's phase, two seconds at most.  A wait that runs out is
// remembered: the CTA waits no more and its states become NaN.
__device__ __forceinline__ bool scan_await(uint64_t* bar, uint32_t parity, volatile bool* lost)
{
    const uint32_t addr = smem_u32(bar);
    if (mbar_try_wait(addr, parity)) return true;
    const uint64_t since = global_timer_ns();
    while (!*lost) {
#pragma unroll 1
        for (int i = 0; i < 32; ++i)
            if (mbar_try_wait(addr, parity)) return true;
        if (global_timer_ns() - since > kScanWaitNs) *lost = true;
    }
    return false;
}

// This lane's elements of an output's rows of 32 V channels from one token on.
template <typename T, int V>
struct ScanOut {
    uint64_t row;
    uint32_t step;
    bool mine;
    __device__ __forceinline__ ScanOut(T* slab, int64_t stride, int64_t t, bool lane_in)
        : row(reinterpret_cast<uint64_t>(slab + t * stride) + threadIdx.x % 32 * (sizeof(T) * V)),
          step(static_cast<uint32_t>(stride) * sizeof(T)),
          mine(lane_in && slab)
    {
    }
    __device__ __forceinline__ void put(int l, Vec<V> v) const
    {
        if (mine) store_pack<T, V, true>(reinterpret_cast<T*>(scan_row(row, step, l)), v.v);
    }
};

// ---- joining ------------------------------------------------------------------------------

// What a warp or a CTA does to the value that enters it: cut ? b : a v + b.
template <int V>
struct ScanMap {
    Vec<V> a, b;
    bool cut;
    __device__ __forceinline__ void clear()
    {
        a = Vec<V>::of(1.0f);
        b = Vec<V>::of(0.0f);
        cut = false;
    }
    // the value is `v` here, whatever entered
    __device__ __forceinline__ void restart(Vec<V> v)
    {
        b = v;
        cut = true;
    }
    __device__ __forceinline__ Vec<V> operator()(Vec<V> v) const
    {
        return cut ? b : vec_fma(a, v, b);
    }
    // this, then `next`
    __device__ __forceinline__ void then(const ScanMap& next)
    {
        b = next(b);
        cut |= next.cut;
        a = a * next.a;
    }
};

// A lane's part of a map on its way through shared memory: one access of 8 V
// bytes.  A factor is never negative, so the sign of a[0] tells that the map cuts.
template <int V>
struct alignas(8 * V) ScanSlot {
    float a[V], b[V];
    __device__ __forceinline__ explicit ScanSlot(const ScanMap<V>& m)
    {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            a[i] = m.a.v[i];
            b[i] = m.b.v[i];
        }
        if (m.cut) a[0] = -a[0];
    }
    __device__ __forceinline__ operator ScanMap<V>() const
    {
        ScanMap<V> m;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            m.a.v[i] = i == 0 ? fabsf(a[i]) : a[i];
            m.b.v[i] = b[i];
        }
        m.cut = __float_as_int(a[0]) < 0;
        return m;
    }
};

// The h map of a warp going backwards, beside its u map, which has the same
// factors: only what it adds, and whether it cuts (uniform in the warp).
template <int V, int K>
struct ScanAdds {
    alignas(16) float b[2][K][32 * V];
    int cut[2][K];
    __device__ __forceinline__ void put(int turn, int k, const ScanMap<V>& m)
    {
        const int lane = threadIdx.x % 32;
#pragma unroll
        for (int i = 0; i < V; ++i) b[turn][k][lane * V + i] = m.b.v[i];
        if (lane == 0) cut[turn][k] = m.cut;
    }
    __device__ __forceinline__ Vec<V> apply(int turn, int k, const ScanMap<V>& u, Vec<V> v) const
    {
        const int lane = threadIdx.x % 32;
        ScanMap<V> m;
        m.a = u.a;
        m.b = vec_of(load_pack<float, V, true>(&b[turn][k][lane * V]));
        m.cut = cut[turn][k];
        return m(v);
    }
};

// Maps of K partners for 32 lanes in shared memory, twice: a segment's writes
// never meet reads of the segment before, which lie a barrier behind.
template <int V, int K>
struct ScanMaps {
    alignas(16) uint8_t bytes[2][K][32 * sizeof(ScanSlot<V>)];
    __device__ __forceinline__ ScanSlot<V>* at(int turn, int k)
    {
        return reinterpret_cast<ScanSlot<V>*>(bytes[turn][k]) + threadIdx.x % 32;
    }
};

// The same for the CTAs of a cluster, with a barrier for each turn that counts
// the bytes which the CTAs (this one too) send.
template <int V, int K>
struct ScanCluster {
    ScanMaps<V, K> maps;
    alignas(8) uint64_t full[2];
};

__device__ __forceinline__ void scan_cluster_sync()
{
    asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;" ::: "memory");
}

template <int V, int K>
__device__ __forceinline__ void scan_cluster_open(ScanCluster<V, K>& s)
{
    if (threadIdx.x == 0) {
        mbar_init(&s.full[0], 1);
        mbar_init(&s.full[1], 1);
        fence_mbarrier_init();
    }
    scan_cluster_sync();  // no CTA sends before all have started and set up their barriers
}

// Lane's slot -> CTA `rank`'s copy of it; the bytes count on that CTA's barrier.
template <int V>
__device__ __forceinline__ void scan_send(ScanSlot<V>* to, uint64_t* bar, int rank, const ScanSlot<V>& v)
{
    uint32_t at, b;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(to)), "r"(rank));
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(smem_u32(bar)), "r"(rank));
    if constexpr (V > 1) {
        static_assert(V == 2, "one vector of four");
        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(at),
                     "f"(v.a[0]), "f"(v.a[1]), "f"(v.b[0]), "f"(v.b[1]), "r"(b)
                     : "memory");
    } else {
        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(at),
                     "f"(v.a[0]), "f"(v.b[0]), "r"(b)
                     : "memory");
    }
}

// Folds `value` (what enters segment k) through the CTAs of the cluster in
// their order, or the reverse, and returns what enters this CTA; afterwards
// `value` is what leaves the segment.  `mine` is the whole CTA's map.  A map's
// slots are written again two segments later, by CTAs that have this CTA's
// map of the segment between, which it sends when all its warps have read.
template <int V, int W, bool REVERSE, int K>
__device__ __forceinline__ void scan_join_cluster(ScanCluster<V, K>& s, int k, int ctas, int rank, const ScanMap<V>& mine,
                                                  Vec<V>& value, Vec<V>& enters, volatile bool* lost)
{
    const int turn = k & 1;
    if (threadIdx.x == 0) mbar_arrive_expect_tx(&s.full[turn], ctas * 32 * sizeof(ScanSlot<V>));
    const ScanSlot<V> slot(mine);
    for (int to = scan_warp(); to < ctas; to += W)
        scan_send<V>(s.maps.at(turn, rank), &s.full[turn], to, slot);
    const bool there = scan_await(&s.full[turn], k >> 1 & 1, lost);
#pragma unroll 2
    for (int n = 0; n < ctas; ++n) {
        const int r = REVERSE ? ctas - 1 - n : n;
        if (r == rank) enters = value;
        value = ScanMap<V>(*s.maps.at(turn, r))(value);
    }
    if (!there) value = enters = Vec<V>::of(__int_as_float(0x7fffffff));
}

// From the warps' maps of a CTA in their order, or the reverse: what all do,
// and what those before this warp do.  `cuts`: one of them may cut.
template <int V, int W, bool REVERSE>
__device__ __forceinline__ void scan_join_warps(ScanMaps<V, W>& maps, int turn, int warp, bool cuts, ScanMap<V>& before,
                                                ScanMap<V>& all)
{
    all.clear();
    before.clear();
    if (cuts) {
#pragma unroll 1
        for (int n = 0; n < W; ++n) {
            const int w = REVERSE ? W - 1 - n : n;
            if (w == warp) before = all;
            all.then(*maps.at(turn, w));
        }
        return;
    }
    ScanMap<V> m[W];
#pragma unroll
    for (int n = 0; n < W; ++n) m[n] = *maps.at(turn, REVERSE ? W - 1 - n : n);
#pragma unroll
    for (int n = 0; n < W; ++n) {
        if (n == (REVERSE ? W - 1 - warp : warp)) {
            before.a = all.a;
            before.b = all.b;
        }
        all.b = vec_fma(m[n].a, all.b, m[n].b);
        all.a = all.a * m[n].a;
    }
}

// The same where the CTA is alone: what enters this warp, and `value` from
// what enters the segment to what leaves it.
template <int V, int W, bool REVERSE>
__device__ __forceinline__ Vec<V> scan_fold_warps(ScanMaps<V, W>& maps, int turn, int warp, bool cuts, Vec<V>& value)
{
    Vec<V> enters = value;
    if (cuts) {
#pragma unroll 1
        for (int n = 0; n < W; ++n) {
            const int w = REVERSE ? W - 1 - n : n;
            if (w == warp) enters = value;
            value = ScanMap<V>(*maps.at(turn, w))(value);
        }
        return enters;
    }
    ScanMap<V> m[W];
#pragma unroll
    for (int n = 0; n < W; ++n) m[n] = *maps.at(turn, REVERSE ? W - 1 - n : n);
#pragma unroll
    for (int n = 0; n < W; ++n) {
        if (n == (REVERSE ? W - 1 - warp : warp)) enters = value;
        value = vec_fma(m[n].a, value, m[n].b);
    }
    return enters;
}

// ---- forwards -------------------------------------------------------------------------------

constexpr int kScanStages = 2;

// A CTA's copies: kScanStages pieces of rows for each of its W warps.
template <int W, bool TMA>
struct ScanFlight {
    alignas(8) uint64_t full[TMA ? kScanStages : 1][W];
    bool lost;  // a wait ran out
    __device__ __forceinline__ void open()
    {
        if (threadIdx.x == 0) {
            lost = false;
            if constexpr (TMA) {
#pragma unroll
                for (int i = 0; i < kScanStages * W; ++i) mbar_init(&full[0][0] + i, 1);
                fence_mbarrier_init();
            }
        }
        __syncthreads();
    }
    // Waits for the warp's piece k.
    __device__ __forceinline__ bool wait(int warp, int k)
    {
        if constexpr (TMA) return scan_await(&full[k % kScanStages][warp], k / kScanStages & 1, &lost);
        scan_wait<kScanStages - 1>();
        return true;
    }
};

struct ScanMapsTma {
    CUtensorMap x, g, d_out;  // [B, T, D] in boxes of 16 rows and 32 V channels
};

template <typename TX, typename TG, int V, int W>
constexpr int scan_forward_smem()
{
    return kScanStages * W * (ScanRows<TX, V, true>::kBytes + ScanRows<TG, V, true>::kBytes);
}

template <typename TX, typename TG, int V, int W, bool TMA>
__global__ void __launch_bounds__(W * 32, 16 / W)
    scan_forward_kernel(const ScanParams p, const __grid_constant__ ScanMapsTma maps)
{
    using RX = ScanRows<TX, V, TMA>;
    using RG = ScanRows<TG, V, TMA>;
    constexpr int kPiece = RX::kBytes + RG::kBytes;
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ ScanMaps<V, W> warps;
    __shared__ ScanCluster<V, kScanForwardCluster> ctas;
    __shared__ ScanFlight<W, TMA> flight;

    const int warp = scan_warp(), lane = threadIdx.x % 32;
    const int rank = blockIdx.x % p.cluster;
    const int64_t slab = static_cast<int64_t>(blockIdx.x / p.cluster) * 32 * V, c = slab + lane * V, b = blockIdx.y;
    const bool mine = c < p.D;
    constexpr int kTile = W * kScanSteps;  // tokens of this CTA in a segment
    const int segments = static_cast<int>((p.T + kTile * p.cluster - 1) / (kTile * p.cluster));
    const int64_t chunks = (p.T + kScanChunk - 1) / kScanChunk;
    ScanBorders seqs(p, false);
    TX* const out = static_cast<TX*>(p.out) + b * p.o_sb + slab;

    auto first_token = [&](int seg) {
        return (static_cast<int64_t>(seg) * p.cluster + rank) * kTile + warp * kScanSteps;
    };
    auto piece = [&](int seg) { return ring + (seg % kScanStages * W + warp) * kPiece; };
    auto fetch = [&](int seg) {
        uint8_t* const to = piece(seg);
        if constexpr (TMA) {
            if (seg < segments) {
                __syncwarp();  // all lanes have read what the piece held
                if (lane == 0) {
                    uint64_t* const full = &flight.full[seg % kScanStages][warp];
                    const int t = static_cast<int>(first_token(seg));
                    mbar_arrive_expect_tx(full, kPiece);
                    RX::fetch_tma(&maps.x, static_cast<int>(slab), t, static_cast<int>(b), full, to);
                    RG::fetch_tma(&maps.g, static_cast<int>(slab), t, static_cast<int>(b), full, to + RX::kBytes);
                }
            }
        } else {
            if (seg < segments && mine) {
                const int64_t t = first_token(seg);
                RX::fetch(static_cast<const TX*>(p.x) + b * p.x_sb + slab, p.x_st, t, p.T, to);
                RG::fetch(static_cast<const TG*>(p.g) + b * p.g_sb + slab, p.g_st, t, p.T, to + RX::kBytes);
            }
            scan_commit();
        }
    };
    flight.open();
#pragma unroll
    for (int s = 0; s < kScanStages; ++s) fetch(s);
    if (p.cluster > 1) scan_cluster_open(ctas);
    if (rank == 0) scan_empty_sequences<V, W>(p, p.h0, p.h0_sn, p.ht, p.ht_sn, c, mine);

    Vec<V> state = Vec<V>::of(0.0f);  // what enters the segment

    for (int seg = 0; seg < segments; ++seg) {
        const int turn = seg & 1;
        const int64_t t = first_token(seg);
        const uint32_t borders = seqs.at<false>(p, b, t), dead = seqs.dead(t);
        const bool plain = (borders | dead) == 0;
        scan_pace(p, seg == 0);
        const bool there = flight.wait(warp, seg);
        const uint8_t *const px = piece(seg), *const pg = px + RX::kBytes;

        Vec<V> a[kScanSteps], x[kScanSteps];
        ScanMap<V> m;
        m.clear();
        if (plain) {
#pragma unroll
            for (int l = 0; l < kScanSteps; ++l) {
                x[l] = vec_of(RX::get(px, l));
                a[l] = vec_exp(vec_of(RG::get(pg, l)));
                m.a = m.a * a[l];
                m.b = vec_fma(a[l], m.b, x[l]);
            }
        } else {
#pragma unroll
            for (int l = 0; l < kScanSteps; ++l) {
                x[l] = vec_of(RX::get(px, l));
                a[l] = vec_exp(vec_of(RG::get(pg, l)));
                if (dead >> l & 1) {  // no sequence's, or no token: the state is 0
                    a[l] = Vec<V>::of(1.0f);
                    x[l] = Vec<V>::of(0.0f);
                    m.restart(x[l]);
                } else if (borders >> l & 1) {
                    m.restart(scan_load_state<V>(p.h0, p.h0_sn, seqs.of(l), c, mine));
                }
                m.a = m.a * a[l];
                m.b = vec_fma(a[l], m.b, x[l]);
            }
        }
        fetch(seg + kScanStages);
        if (!there) m.b = Vec<V>::of(__int_as_float(0x7fffffff));

        *warps.at(turn, warp) = ScanSlot<V>(m);
        const bool cuts = __syncthreads_or(m.cut);
        Vec<V> h;
        if (p.cluster == 1) {
            h = scan_fold_warps<V, W, false>(warps, turn, warp, cuts, state);
        } else {
            ScanMap<V> before, all;
            scan_join_warps<V, W, false>(warps, turn, warp, cuts, before, all);
            scan_join_cluster<V, W, false>(ctas, seg, p.cluster, rank, all, state, h, &flight.lost);
            h = before(h);
        }

        if (p.chunk && warp == 0 && t % kScanChunk == 0 && t < p.T)
            scan_store_state<V>(p.chunk, p.D, b * chunks + t / kScanChunk, c, mine, h);
        const ScanOut<TX, V> to(out, p.o_st, t, mine);
        if (plain) {
#pragma unroll
            for (int l = 0; l < kScanSteps; ++l) {
                h = vec_fma(a[l], h, x[l]);
                to.put(l, h);
            }
        } else {
#pragma unroll
            for (int l = 0; l < kScanSteps; ++l) {
                const bool out_of = dead >> l & 1;
                if (out_of) h = Vec<V>::of(0.0f);
                else if (borders >> l & 1) h = scan_load_state<V>(p.h0, p.h0_sn, seqs.of(l), c, mine);
                h = vec_fma(a[l], h, x[l]);
                if (t + l < p.T) to.put(l, h);
                if (!out_of && p.ht && (borders >> (l + 1) & 1))
                    scan_store_state<V>(p.ht, p.ht_sn, seqs.of(l), c, mine, h);
            }
        }
    }
    scan_pace_end(p);
    if (p.cluster > 1) scan_cluster_sync();  // none leaves while another may still send to it
}

// ---- backwards --------------------------------------------------------------------------------

template <typename TX, typename TG, int V, int W>
constexpr int scan_backward_smem()
{
    return kScanStages * W * (2 * ScanRows<TX, V, true>::kBytes + ScanRows<TG, V, true>::kBytes);
}

template <typename TX, typename TG, int V, int W, bool TMA>
__global__ void __launch_bounds__(W * 32, 16 / W)
    scan_backward_kernel(const ScanParams p, const __grid_constant__ ScanMapsTma maps)
{
    using RX = ScanRows<TX, V, TMA>;
    using RG = ScanRows<TG, V, TMA>;
    constexpr int kPiece = 2 * RX::kBytes + RG::kBytes;
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ ScanMaps<V, W> warps_u;
    __shared__ ScanAdds<V, W> warps_h;
    __shared__ ScanCluster<V, kScanBackwardCluster> ctas;
    __shared__ ScanFlight<W, TMA> flight;

    const int warp = scan_warp(), lane = threadIdx.x % 32;
    const int rank = blockIdx.x % p.cluster;
    const int64_t slab = static_cast<int64_t>(blockIdx.x / p.cluster) * 32 * V, c = slab + lane * V, b = blockIdx.y;
    const bool mine = c < p.D;
    constexpr int kTile = W * kScanSteps;  // tokens of this CTA in a segment
    const int segments = static_cast<int>((p.T + kTile * p.cluster - 1) / (kTile * p.cluster));
    const int64_t chunks = (p.T + kScanChunk - 1) / kScanChunk;
    ScanBorders seqs(p, true);
    TX* const dx = p.dx ? static_cast<TX*>(p.dx) + b * p.dx_sb + slab : nullptr;
    TG* const dg = p.dg ? static_cast<TG*>(p.dg) + b * p.dg_sb + slab : nullptr;

    // segments run from the last to the first: turn k is segment segments - 1 - k
    auto first_token = [&](int k) {
        return (static_cast<int64_t>(segments - 1 - k) * p.cluster + rank) * kTile + warp * kScanSteps;
    };
    auto piece = [&](int k) { return ring + (k % kScanStages * W + warp) * kPiece; };
    auto fetch = [&](int k) {
        uint8_t* const to = piece(k);
        if constexpr (TMA) {
            if (k < segments) {
                __syncwarp();
                if (lane == 0) {
                    uint64_t* const full = &flight.full[k % kScanStages][warp];
                    const int t = static_cast<int>(first_token(k));
                    mbar_arrive_expect_tx(full, p.d_out ? kPiece : kPiece - RX::kBytes);
                    RX::fetch_tma(&maps.x, static_cast<int>(slab), t, static_cast<int>(b), full, to);
                    RG::fetch_tma(&maps.g, static_cast<int>(slab), t, static_cast<int>(b), full, to + RX::kBytes);
                    if (p.d_out)
                        RX::fetch_tma(&maps.d_out, static_cast<int>(slab), t, static_cast<int>(b), full,
                                      to + RX::kBytes + RG::kBytes);
                }
            }
        } else {
            if (k < segments && mine) {
                const int64_t t = first_token(k);
                RX::fetch(static_cast<const TX*>(p.x) + b * p.x_sb + slab, p.x_st, t, p.T, to);
                RG::fetch(static_cast<const TG*>(p.g) + b * p.g_sb + slab, p.g_st, t, p.T, to + RX::kBytes);
                if (p.d_out)
                    RX::fetch(static_cast<const TX*>(p.d_out) + b * p.do_sb + slab, p.do_st, t, p.T,
                              to + RX::kBytes + RG::kBytes);
            }
            scan_commit();
        }
    };
    flight.open();
#pragma unroll
    for (int s = 0; s < kScanStages; ++s) fetch(s);
    if (p.cluster > 1) scan_cluster_open(ctas);
    if (rank == 0) scan_empty_sequences<V, W>(p, p.d_ht, p.dht_sn, p.d_h0, p.dh0_sn, c, mine);

    Vec<V> enter = Vec<V>::of(0.0f);  // u that enters the segment from the right

    for (int k = 0; k < segments; ++k) {
        const int turn = k & 1;
        const int64_t t = first_token(k);
        const uint32_t borders = seqs.at<true>(p, b, t), dead = seqs.dead(t);
        const bool plain = (borders | dead) == 0;
        const int64_t chunk = t / kScanChunk;
        Vec<V> h = scan_load_state<V>(p.chunk, p.D, b * chunks + chunk, c, mine && chunk < chunks);  // before this CTA's tokens
        scan_pace(p, k == 0);
        const bool there = flight.wait(warp, k);
        const uint8_t *const px = piece(k), *const pg = px + RX::kBytes, *const pd = pg + RG::kBytes;
        auto get_x = [&](int l) { return vec_of(RX::get(px, l)); };
        auto get_a = [&](int l) { return vec_exp(vec_of(RG::get(pg, l))); };
        auto get_d = [&](int l) { return vec_of(p.d_out ? RX::get(pd, l) : pack_zero<TX, V>()); };

        // u leaves as A u + sum over l of (a_0 .. a_l) d_l, so both maps come of
        // one walk; x and d_out are read again from shared memory afterwards
        // rather than kept, which leaves registers for twice the warps
        Vec<V> a[kScanSteps];
        ScanMap<V> mh, mu;
        mh.clear();
        mu.clear();
        if (plain) {
#pragma unroll
            for (int l = 0; l < kScanSteps; ++l) {
                a[l] = get_a(l);
                mh.a = mh.a * a[l];
                mh.b = vec_fma(a[l], mh.b, get_x(l));
                if (p.d_out) mu.b = vec_fma(mh.a, get_d(l), mu.b);
            }
        } else {
#pragma unroll
            for (int l = 0; l < kScanSteps; ++l) {
                a[l] = get_a(l);
                if (dead >> l & 1) {
                    a[l] = Vec<V>::of(1.0f);
                    mh.restart(Vec<V>::of(0.0f));
                    mu.cut = true;
                    continue;
                }
                if (borders >> l & 1) mh.restart(scan_load_state<V>(p.h0, p.h0_sn, seqs.of(l), c, mine));
                mh.a = mh.a * a[l];
                mh.b = vec_fma(a[l], mh.b, get_x(l));
                if (!mu.cut) {  // what lies right of the first sequence's end does not reach out
                    mu.b = vec_fma(mh.a, get_d(l), mu.b);
                    if (borders >> (l + 1) & 1) {
                        mu.b = vec_fma(mh.a, scan_load_state<V>(p.d_ht, p.dht_sn, seqs.of(l), c, mine), mu.b);
                        mu.cut = true;
                    }
                }
            }
        }
        mu.a = mh.a;
        if (!there) mh.b = mu.b = Vec<V>::of(__int_as_float(0x7fffffff));

        warps_h.put(turn, warp, mh);
        *warps_u.at(turn, warp) = ScanSlot<V>(mu);
        const bool cuts = __syncthreads_or(mh.cut || mu.cut);
#pragma unroll 1
        for (int w = 0; w < warp; ++w) h = warps_h.apply(turn, w, *warps_u.at(turn, w), h);
        Vec<V> u;
        if (p.cluster == 1) {
            u = scan_fold_warps<V, W, true>(warps_u, turn, warp, cuts, enter);
        } else {
            ScanMap<V> after, all;
            scan_join_warps<V, W, true>(warps_u, turn, warp, cuts, after, all);
            scan_join_cluster<V, W, true>(ctas, k, p.cluster, rank, all, enter, u, &flight.lost);
            u = after(u);
        }

        const ScanOut<TX, V> to_x(dx, p.dx_st, t, mine);
        const ScanOut<TG, V> to_g(dg, p.dg_st, t, mine);
        Vec<V> before[kScanSteps];  // h_{t-1}
        if (plain) {
#pragma unroll
            for (int l = 0; l < kScanSteps; ++l) {
                before[l] = h;
                h = vec_fma(a[l], h, get_x(l));
            }
#pragma unroll
            for (int l = kScanSteps - 1; l >= 0; --l) {
                const Vec<V> dh = p.d_out ? u + get_d(l) : u;
                u = a[l] * dh;
                to_x.put(l, dh);
                to_g.put(l, u * before[l]);
            }
        } else {
#pragma unroll
            for (int l = 0; l < kScanSteps; ++l) {
                before[l] = h;
                if (dead >> l & 1) continue;
                if (borders >> l & 1) before[l] = scan_load_state<V>(p.h0, p.h0_sn, seqs.of(l), c, mine);
                h = vec_fma(a[l], before[l], get_x(l));
            }
#pragma unroll
            for (int l = kScanSteps - 1; l >= 0; --l) {
                Vec<V> dh = Vec<V>::of(0.0f), dgv = dh;
                if (dead >> l & 1) {
                    u = dh;
                } else {
                    if (borders >> (l + 1) & 1) u = scan_load_state<V>(p.d_ht, p.dht_sn, seqs.of(l), c, mine);
                    dh = u + get_d(l);
                    u = a[l] * dh;
                    dgv = u * before[l];
                    if (p.d_h0 && (borders >> l & 1))
                        scan_store_state<V>(p.d_h0, p.dh0_sn, seqs.of(l), c, mine, u);
                }
                if (t + l < p.T) {
                    to_x.put(l, dh);
                    to_g.put(l, dgv);
                }
            }
        }
        fetch(k + kScanStages);
    }
    scan_pace_end(p);
    if (p.cluster > 1) scan_cluster_sync();
}

}  // namespace cgdr
