// The shared prefixes of larger groups: attention of up to 256 query rows (requests of the group times the query heads
// of a cache head) against a range of the prefix's keys, on the tcgen05 tensor cores.
//
// With r rows a key and its value (4 D bytes) are used for 4 D r operations: above 258 rows the multiplications bound
// the work on this GPU, and already at 32 rows the split kernel's reading of the keys once per 16 rows would.
//
// A block of kKeys = 128 keys is a unit.  Two streams of 128 rows each go through the units of an item:
//     S[128, 128] = Q K^T            tcgen05.mma, Q and K from shared memory
//     P = 2^(scale S - m)            by the stream's four warps, a thread per row, S from and P (16 bits) to TMEM
//     O[128, D] += P V               tcgen05.mma, P from TMEM, V from shared memory (its rows are the contraction)
// While the warps of one stream compute exponentials, the tensor core multiplies for the other.  Where an item has more
// than 128 rows the streams hold different rows and share each block; else they hold the same rows and take the blocks in
// turns, and each leaves a part of its own.
//
// The running maximum is not followed exactly: the sums are only rescaled when a row's maximum has grown by more than
// 2^8, since fp32 sums and 16-bit weights up to 256 lose nothing by a common factor.  P is rounded to the 16-bit type
// (by up to 2^-8 or 2^-11 of its size, as often up as down): what the output's own rounding does again.  The sum of the weights
// takes them as they were, so lse does not feel that rounding and a row's weights sum to one only up to it.
//
// Warps 0..3 and 4..7: the streams.  Warp 8: one thread issues the multiplications.  Warps 9..11 bring keys and values
// into a ring of blocks by asynchronous 16-byte copies in the 128-byte swizzled layout the multiplications read, page
// by page, whatever the page size, with zeros in place of keys behind the prefix or in pages that do not exist.
//
// The split kernel, which does the rest of a call, runs behind this one: both want all of an SM's shared memory, and what it reads is
// only sure to be seen after a wait of its own.  (Side by side, on SMs shared out by their work and without that wait, the three larger
// calls took 2 to 9 % less: 307, 68 and 120 us instead of 312, 72 and 132 us.)
//
// 256 requests of 64 heads over 8 of 128, a prefix of 16384 tokens: a unit of 256 rows takes an SM some 4500 cycles, of which the
// multiplications need 2048 and the exponentials of a stream's warps 1500, while each waits for the other's result twice: 0.83
// PFLOP/s over the whole GPU, half of what a library product reaches.  64 requests, a prefix of 8192: 55 us of which 12 are start and
// end (queries, TMEM, the partial rows).  Tried and taken back: two threads a row (half the row each, no registers for more
// in flight: 328 us against 314 us in all), scores kept in registers (spills: 587 us against 325 us).
//
// Every wait is bounded: on expiry the outputs become NaN and `status` says so (tc_common.cuh).
#include <type_traits>

#include "attn_common.cuh"
#include "tc_common.cuh"

namespace b200lora {

namespace {

constexpr int kStreamRows = kTcRows;
constexpr int kThreads = 384;
constexpr int kCopyWarps = 3;
constexpr int kCopyThreads = kCopyWarps * 32;
constexpr float kSlack = 8.f;                     // in powers of two

template <int D, int RING> struct Wide {
    static constexpr int kQ = kStreamRows * D * 2;           // a stream's queries
    static constexpr int kBlock = kWideKeys * D * 2;         // keys or values of a unit
    static constexpr int kBytes = 2 * kQ + RING * kBlock;
};
constexpr int kMaxRing = 8;
constexpr int kMissing = 16;                      // more blocks of keys than can lie between their copies and their use
struct WideShared {
    uint4 missing[kMissing][kCopyWarps];          // keys of a block in pages that do not exist, as each copy warp saw them
    unsigned long long full[kMaxRing], empty[kMaxRing], q_ready[2], s_full[2], p_ready[2], o_full[2];
    unsigned long long warp_sum[kThreads / 32];
    unsigned long long drained;
    unsigned tmem, err;
    int bad, pad[3];
};
static_assert(sizeof(WideShared) % 16 == 0, "the scan's arrays follow");

// one of the barrier's arrivals, once this thread's copies so far have landed
__device__ __forceinline__ void arrive_when_copied(unsigned b) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(b) : "memory");
}
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// An item's part of a worker: blocks [b0, b0 + n) of tile `tile` of cache head `h` of group `g`.
struct Part {
    int g, h, tile, b0, n, rows, first, keys;
    bool dual;             // the streams hold different rows
    size_t slot;           // first row of the part's partial results
};

__device__ __forceinline__ Part part_of(const AttnParams& p, const int* su, const int* st, bool usable, long long u, long long u_end) {
    Part t;
    int ignored = 0;
    const int n_kv = p.c.n_kv_heads;
    const int uh = (int)quotient(u, n_kv);
    t.g = entity_at(su, p.a.n_groups, uh);
    const Entity e = group_of<kWideRows, kWideKeys, true>(p, t.g, usable, ignored);
    const int per_head = e.tiles * e.chunks;
    const long long of_entity = u - (long long)n_kv * su[t.g];
    t.h = (int)quotient(of_entity, per_head);
    const int rest = (int)(of_entity - (long long)t.h * per_head);
    t.tile = rest / e.chunks;
    t.b0 = rest - t.tile * e.chunks;
    t.n = (int)min((long long)(e.chunks - t.b0), u_end - u);
    t.rows = min(kWideRows, e.rows - t.tile * kWideRows);
    t.first = e.first;
    t.keys = e.keys;
    t.dual = t.rows > kStreamRows;
    t.slot = attn_group_rows(p) + attn_request_rows(p) + ((size_t)n_kv * st[t.g] + (size_t)t.h * e.tiles + t.tile + blockIdx.x) * kWideRows;
    return t;
}

template <typename T, int D, int RING>
__global__ void __launch_bounds__(kThreads, 1) attn_wide_kernel(const __grid_constant__ AttnParams p) {
    extern __shared__ unsigned char smem_raw[];
    using W = Wide<D, RING>;
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    WideShared& sh = *reinterpret_cast<WideShared*>(smem + W::kBytes);
    int* su = reinterpret_cast<int*>(&sh + 1);
    int* st = su + p.a.n_groups + 1;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto bar = [](unsigned long long& b) { return smem_u32(&b); };
    unsigned* err = &sh.err;

    pdl_wait_prior();
    if (tid == 0) pdl_launch_dependents();       // (before TMEM: the split kernel, which follows, takes none)
    if (tid < kMaxRing) {
        if (tid < RING) { mbar_init(bar(sh.full[tid]), kCopyThreads + kCopyWarps); mbar_init(bar(sh.empty[tid]), 1); }
        if (tid < 2) {
            mbar_init(bar(sh.q_ready[tid]), kStreamRows);
            mbar_init(bar(sh.p_ready[tid]), kStreamRows);
            mbar_init(bar(sh.s_full[tid]), 1);
            mbar_init(bar(sh.o_full[tid]), 1);
        }
        if (tid == 0) mbar_init(bar(sh.drained), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) tmem_alloc(smem_u32(&sh.tmem));
    if (tid == 0) { sh.err = 0u; sh.bad = 0; }
    __syncthreads();
    const int n_g = p.a.n_groups, n_kv = p.c.n_kv_heads;
    const bool usable = scan_units<kThreads>(n_g, n_g, su, st, sh.warp_sum, &sh.bad, [&](int e, bool ok, int& bad) {
        const Entity t = group_of<kWideRows, kWideKeys, true>(p, e, ok, bad);
        return ((unsigned long long)t.tiles << 32) | (unsigned)(t.tiles * t.chunks);
    });
    if (blockIdx.x == 0)
        for (int i = tid; i <= n_g; i += kThreads) { p.wide_units[i] = su[i]; p.wide_tile[i] = st[i]; }
    const long long total = (long long)su[n_g] * n_kv;
    const int workers = (int)min((long long)gridDim.x, total);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = *reinterpret_cast<volatile unsigned*>(&sh.tmem);
    if ((int)blockIdx.x >= workers) {
        if (warp == 8) tmem_dealloc(tmem);
        return;
    }
    const long long u_first = unit_of_worker(total, blockIdx.x, workers), u_end = unit_of_worker(total, blockIdx.x + 1, workers);
    auto part_at = [&](long long u) { return part_of(p, su, st, usable, u, u_end); };

    const unsigned ring = smem_u32(smem) + 2 * W::kQ;
    // The ring's order within a part: where the streams share blocks, K0 V0 K1 V1 ...; where they take them in turns,
    // K0 K1 V0 K2 V1 K3 ...: what the multiplications need next always comes next.
    if (warp >= 9) {
        // ================= copies =================
        const int cw = warp - 9;
        constexpr int kPieces = D / 8, kRowsAt = 32 / kPieces;
        constexpr int kGroups = kWideKeys / kRowsAt, kMine = (kGroups + kCopyWarps - 1) / kCopyWarps;   // a copy's rows; this warp's copies
        static_assert(kMine * kRowsAt <= 64, "two rows' places a lane");
        const int piece = lane % kPieces, sub = lane / kPieces;
        const int in_page = (1 << p.page_shift) - 1;
        unsigned n = 0, n_keys = 0;              // blocks, and blocks of keys, so far
        // The places of the rows that this warp copies, one or two a lane: row i is row i % kRowsAt of its copy i / kRowsAt.
        // The page table is read a block ahead, or each copy would wait for it.
        auto row_of = [&](int i) { return (cw + kCopyWarps * (i / kRowsAt)) * kRowsAt + i % kRowsAt; };
        int page[2];
        bool fine = true;                        // no wait of this warp has expired
        for (long long u = u_first; u < u_end && fine;) {
            const Part t = part_at(u);
            const int* table = p.a.prefix_table + (long long)t.g * p.a.prefix_table_row;
            auto block_at = [&](int i, bool& is_v) {
                if (t.dual) { is_v = i & 1; return i >> 1; }
                const int lead = min(2, t.n), j = i - lead, pairs = max(t.n - 2, 0);
                if (j < 0) { is_v = false; return i; }
                if (j < 2 * pairs) { is_v = !(j & 1); return is_v ? j >> 1 : (j >> 1) + 2; }
                is_v = true;
                return j - pairs;
            };
            auto read_table = [&](int b) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int row = row_of(lane + 32 * k), key = (t.b0 + b) * kWideKeys + row;
                    page[k] = row < kWideKeys && key < t.keys ? __ldg(table + (key >> p.page_shift)) : kNoPage;
                }
            };
            bool is_v, next_v;
            int b = block_at(0, is_v);
            read_table(b);
            for (int i = 0; i < 2 * t.n; ++i, ++n) {
                if (u == u_first && i == 1) {    // the first multiplication needs the queries and one block: the others wait for those
                    for (int q = 0; q < 2; ++q)
                        if (t.dual || q < t.n) fine = fine && mbar_reached(bar(sh.q_ready[q]), 0, err, 7);
                }
                const int slot = n % RING;
                fine = fine && mbar_reached(bar(sh.empty[slot]), ((n / RING) & 1) ^ 1, err, 1);
                fine = __all_sync(0xffffffffu, fine);
                if (!fine) break;
                long long at[2];                 // < 0: zeros
                bool lost[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int row = row_of(lane + 32 * k), key = (t.b0 + b) * kWideKeys + row;
                    const bool fine = (unsigned)page[k] < (unsigned)p.c.n_pages;
                    lost[k] = !fine && row < kWideKeys && key < t.keys;
                    at[k] = fine ? (long long)page[k] * p.c.page_stride + (long long)(key & in_page) * p.c.token_stride : -1;
                }
                if (!is_v) {
                    uint4 missing = make_uint4(0u, 0u, 0u, 0u);
                    if (__any_sync(0xffffffffu, lost[0] || lost[1])) {
                        if (lane == 0 && p.a.status) atomicOr(p.a.status, B200_DECODE_BAD_PAGE);
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const int row = row_of(lane + 32 * k);
                            const unsigned bit = lost[k] ? 1u << (row & 31) : 0u;
                            missing.x |= row >> 5 == 0 ? bit : 0u; missing.y |= row >> 5 == 1 ? bit : 0u;
                            missing.z |= row >> 5 == 2 ? bit : 0u; missing.w |= row >> 5 == 3 ? bit : 0u;
                        }
                        missing.x = __reduce_or_sync(0xffffffffu, missing.x); missing.y = __reduce_or_sync(0xffffffffu, missing.y);
                        missing.z = __reduce_or_sync(0xffffffffu, missing.z); missing.w = __reduce_or_sync(0xffffffffu, missing.w);
                    }
                    if (lane == 0) sh.missing[n_keys % kMissing][cw] = missing;
                    ++n_keys;
                }
                int next = 0;
                if (i + 1 < 2 * t.n) {
                    next = block_at(i + 1, next_v);
                    read_table(next);
                }
                const unsigned dst = ring + slot * W::kBlock;
                const T* base = static_cast<const T*>(is_v ? p.c.v : p.c.k) + (long long)t.h * p.c.head_stride + piece * 8;
#pragma unroll
                for (int j = 0; j < kMine; ++j) {
                    const int g = cw + kCopyWarps * j, row = g * kRowsAt + sub;
                    const long long from = __shfl_sync(0xffffffffu, at[j * kRowsAt >= 32], (j * kRowsAt + sub) & 31);
                    if (g < kGroups) cp_async16(swizzled(dst, row, piece), base + max(from, 0ll), from >= 0);
                }
                arrive_when_copied(bar(sh.full[slot]));
                if (lane == 0) mbar_arrive(bar(sh.full[slot]));  // (for what it wrote by itself: the missing keys)
                b = next;
                is_v = next_v;
            }
            u += t.n;
        }
        cp_wait_all();
        if (cw == 0)                             // nobody else waits for the last blocks' arrivals here
            for (unsigned i = n > RING ? n - RING : 0; i < n; ++i) fine = fine && mbar_reached(bar(sh.empty[i % RING]), (i / RING) & 1, err, 1);
    } else if (warp == 8) {
        // ================= multiplications: one thread =================
        if (lane == 0) {
            const unsigned id_s = idesc_of(Cvt<T>::is_bf16, kWideKeys, false), id_o = idesc_of(Cvt<T>::is_bf16, D, true);
            const unsigned q_low = desc_low(smem_u32(smem), kRowsAreRows), full0 = bar(sh.full[0]), empty0 = bar(sh.empty[0]);
            const unsigned q0 = bar(sh.q_ready[0]), s0 = bar(sh.s_full[0]), p0 = bar(sh.p_ready[0]), o0 = bar(sh.o_full[0]);
            unsigned slot = 0, phase = 0;                        // of the block that is needed next: the ring's order is theirs
            unsigned q_phase = 0, p_phase = 0;                   // bit s: of stream s
            bool fine = true;                                    // no wait has expired
            auto next_block = [&]() {                            // waits for it and returns its slot
                const unsigned at = slot;
                fine = fine && mbar_reached(full0 + at * 8, phase, err, 2);
                fence_async_proxy();                             // the copies wrote through the generic proxy
                if (++slot == RING) { slot = 0; phase ^= 1; }
                return at;
            };
            auto scores = [&](int s, unsigned k, bool last_use) {
                if (!fine) return;
                tc_fence_after();
                const unsigned qa = q_low + s * (W::kQ >> 4), ka = desc_low(ring + k * W::kBlock, kRowsAreRows), d = tmem + s * 128;
                mma_ss<false>(d, qa, ka, id_s);
#pragma unroll
                for (int i = 1; i < D / 16; ++i) {
                    const unsigned off = ((i >> 2) * kPanel + (i & 3) * 32) >> 4;
                    mma_ss<true>(d, qa + off, ka + off, id_s);
                }
                tc_commit(s0 + s * 8);
                if (last_use) tc_commit(empty0 + k * 8);
            };
            auto queries = [&](int s) { fine = fine && mbar_reached(q0 + s * 8, q_phase >> s & 1, err, 3); q_phase ^= 1u << s; };
            auto weigh = [&](int s, unsigned v, bool first, bool last, bool last_use) {
                fine = fine && mbar_reached(p0 + s * 8, p_phase >> s & 1, err, 4);
                p_phase ^= 1u << s;
                if (!fine) return;
                tc_fence_after();
                const unsigned va = desc_low(ring + v * W::kBlock, kRowsAreDepth), d = tmem + 256 + s * 128, w = tmem + s * 128;
                mma_ts(d, w, va, id_o, !first);
#pragma unroll
                for (int i = 1; i < kWideKeys / 16; ++i) mma_ts(d, w + i * 8, va + i * (2048 >> 4), id_o, 1);
                if (last) tc_commit(o0 + s * 8);
                if (last_use) tc_commit(empty0 + v * 8);
            };
            for (long long u = u_first; u < u_end;) {
                const Part t = part_at(u);
                const int n = t.n;
                if (t.dual) {
                    unsigned k = next_block();
                    for (int s = 0; s < 2; ++s) { queries(s); scores(s, k, s == 1); }
                    for (int b = 0; b < n; ++b) {
                        const unsigned v = next_block();
                        const bool more = b + 1 < n;
                        weigh(0, v, b == 0, !more, false);
                        if (more) { k = next_block(); scores(0, k, false); }
                        weigh(1, v, b == 0, !more, true);
                        if (more) scores(1, k, true);
                    }
                } else {
                    for (int s = 0; s < 2 && s < n; ++s) { queries(s); scores(s, next_block(), true); }
                    for (int b = 0; b < n; ++b) {
                        const bool more = b + 2 < n;
                        weigh(b & 1, next_block(), b < 2, !more, true);
                        if (more) scores(b & 1, next_block(), true);
                    }
                }
                u += n;
            }
        }
        __syncwarp();
    } else {
        // ================= the streams =================
        const int s = warp >> 2, row = tid & 127;
        const unsigned lanes = (unsigned)((warp & 3) * 32) << 16;
        const unsigned s_tm = tmem + lanes + s * 128, o_tm = tmem + lanes + 256 + s * 128;
        auto stream_sync = [&]() {
            if (s == 0) asm volatile("bar.sync 1, %0;" ::"n"(kStreamRows) : "memory");
            else asm volatile("bar.sync 2, %0;" ::"n"(kStreamRows) : "memory");
        };
        // scores are compared as they come from the multiplication: a negative scale goes into the queries' signs
        const unsigned flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;
        const float scale = fabsf(p.scale_log2);
        const float kLift = std::is_same_v<T, __half> ? 7.f : 0.f;     // fp16 weights up to 2^(8 + 7), far from its smallest numbers
        unsigned rounds = 0, outs = 0, n_keys = 0;
        bool fine = true;                                        // no wait of this thread has expired
        for (long long u = u_first; u < u_end;) {
            const Part t = part_at(u);
            const int r_in = t.dual ? s * kStreamRows + row : row;
            const bool live = r_in < t.rows;
            const int step = t.dual ? 1 : 2, b_first = t.dual ? 0 : s;
            // ---- queries to shared memory (the stream's last multiplication that reads them is complete)
            if (b_first < t.n) {
                const unsigned qa = smem_u32(smem) + s * W::kQ;
                constexpr int kPieces = D / 8, kBatch = kPieces;
                const int c = row % kPieces;
#pragma unroll
                for (int i0 = 0; i0 < kPieces; i0 += kBatch) {
                    uint4 v[kBatch];
#pragma unroll
                    for (int i = 0; i < kBatch; ++i) {           // neighbouring lanes read neighbouring pieces of a row
                        const int r = ((i0 + i) * kStreamRows + row) / kPieces, in_tile = t.dual ? s * kStreamRows + r : r;
                        v[i] = make_uint4(flip, flip, flip, flip);
                        if (in_tile < t.rows) {
                            const int ra = t.tile * kWideRows + in_tile, request = request_of_row(p, ra);
                            v[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.a.q) + (long long)(t.first + request) * p.a.q_row +
                                                                    (long long)(t.h * p.per + ra - request * p.per) * p.a.q_head + c * 8);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < kBatch; ++i)
                        sts16(swizzled(qa, ((i0 + i) * kStreamRows + row) / kPieces, c), v[i].x ^ flip, v[i].y ^ flip, v[i].z ^ flip, v[i].w ^ flip);
                }
                fence_async_proxy();
                if (fine) mbar_arrive(bar(sh.q_ready[s]));
            }
            const bool warp_live = __ballot_sync(0xffffffffu, live) != 0u;
            float m = -INFINITY, l = 0.f;                        // sums are relative to 2^(m - kLift)
            for (int b = b_first; b < t.n; b += step, ++rounds) {
                fine = fine && mbar_reached(bar(sh.s_full[s]), rounds & 1, err, 5);
                __syncwarp();                                    // lanes may leave a wait one by one: what follows is for whole warps
                tc_fence_after();
                if (warp_live) {
                    // keys behind the prefix, or in pages that do not exist
                    const uint4* lost = sh.missing[(n_keys + b) % kMissing];
                    const uint4 w0 = lost[0], w1 = lost[1], w2 = lost[2];
                    const int valid = t.keys - (t.b0 + b) * kWideKeys;
                    const unsigned gone[4] = {w0.x | w1.x | w2.x, w0.y | w1.y | w2.y, w0.z | w1.z | w2.z, w0.w | w1.w | w2.w};
                    const bool masked = valid < kWideKeys || (gone[0] | gone[1] | gone[2] | gone[3]);
                    auto mask = [&](unsigned (&z)[32], int c) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (c * 32 + j >= valid || (gone[c] >> j & 1u)) z[j] = 0xff800000u;      // -infinity
                    };
                    // The scores are read twice, 32 at a time, for their maximum and for the weights: a row of them would
                    // leave no registers.
                    float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int c = 0; c < 4; c += 2) {
                        unsigned za[32], zb[32];
                        tc_ld32(s_tm + c * 32, za);
                        tc_ld32(s_tm + c * 32 + 32, zb);
                        tc_wait_ld();
                        if (masked) { mask(za, c); mask(zb, c + 1); }
#pragma unroll
                        for (int j = 0; j < 32; ++j) x[j & 3] = fmaxf(fmaxf(x[j & 3], __uint_as_float(za[j])), __uint_as_float(zb[j]));
                    }
                    const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) * scale;
                    if (b == b_first) m = top;
                    else {
                        const bool grown = top > m + kSlack || (m == -INFINITY && top > m);
                        if (__any_sync(0xffffffffu, grown)) {
                            const float f = grown ? (m == -INFINITY ? 0.f : ex2(m - top)) : 1.f;
                            if (grown) m = top;
                            l *= f;
#pragma unroll
                            for (int c = 0; c < D / 32; ++c) {
                                unsigned o[32];
                                tc_ld32(o_tm + c * 32, o);
                                tc_wait_ld();
#pragma unroll
                                for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                                tc_st32(o_tm + c * 32, o);
                            }
                            tc_wait_st();
                        }
                    }
                    const float ref = m == -INFINITY ? 0.f : m - kLift;      // nothing yet: every weight is 0
                    const unsigned long long scale2 = pair(scale, scale), ref2 = pair(-ref, -ref);
                    unsigned long long sum[2] = {0ull, 0ull};
                    unsigned z[2][32];
                    tc_ld32(s_tm, z[0]);
                    tc_wait_ld();
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        // the weights' words lie where the scores of the first half lay: read what is still needed first
                        if (c < 3) tc_ld32(s_tm + (c + 1) * 32, z[(c + 1) & 1]);
                        if (masked) mask(z[c & 1], c);
                        unsigned w[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            float2 e = unpair(fma2(pair(__uint_as_float(z[c & 1][2 * j]), __uint_as_float(z[c & 1][2 * j + 1])), scale2, ref2));
                            e.x = ex2(e.x);
                            e.y = ex2(e.y);
                            sum[j & 1] = add2(sum[j & 1], pair(e.x, e.y));
                            w[j] = Cvt<T>::pack2(e.x, e.y);
                        }
                        if (c < 3) tc_wait_ld();
                        tc_st16(s_tm + c * 16, w);
                    }
                    const float2 sums = unpair(add2(sum[0], sum[1]));
                    l += sums.x + sums.y;
                    tc_wait_st();
                }
                tc_fence_before();
                if (fine) mbar_arrive(bar(sh.p_ready[s]));
            }
            // ---- this worker's part of the rows
            const size_t out_row = t.slot + s * kStreamRows + row;
            if (b_first < t.n) {
                fine = fine && mbar_reached(bar(sh.o_full[s]), outs & 1, err, 6);
                ++outs;
                __syncwarp();
                tc_fence_after();
                // Rows go out through the place of the queries, half a row of each at a time: by themselves the lanes' rows lie D words
                // apart, and every 16 bytes would be a transfer of their own.
                const unsigned at = smem_u32(smem) + s * W::kQ;
                constexpr int kPieces = D / 8;                   // of 16 bytes, of half a row
                const int c_out = row % kPieces;
#pragma unroll
                for (int turn = 0; turn < 2; ++turn) {
                    if (warp_live) {
#pragma unroll
                        for (int c = 0; c < D / 64; ++c) {
                            unsigned o[32];
                            tc_ld32(o_tm + turn * (D / 2) + c * 32, o);
                            tc_wait_ld();
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                sts16(at + row * (D * 2) + (((c * 8 + j) ^ (row & 7)) << 4), o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
                        }
                        tc_fence_before();
                    }
                    stream_sync();
#pragma unroll 4
                    for (int i = 0; i < kPieces; ++i) {
                        const int r = (i * kStreamRows + row) / kPieces, in_tile = t.dual ? s * kStreamRows + r : r;
                        unsigned w[4];
                        lds16(at + r * (D * 2) + ((c_out ^ (r & 7)) << 4), w);
                        if (in_tile < t.rows)
                            reinterpret_cast<uint4*>(p.part + (t.slot + s * kStreamRows + r) * D + turn * (D / 2))[c_out] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    stream_sync();
                }
                if (live) p.part_ml[out_row] = make_float2(m == -INFINITY ? m : m - kLift, l);
            } else if (live) p.part_ml[out_row] = make_float2(-INFINITY, 0.f);
            n_keys += t.n;
            u += t.n;
        }
    }
    tc_fence_before();
    __syncthreads();
    const bool lost = *reinterpret_cast<volatile unsigned*>(err) != 0u;
    if (warp == 8) {
        if (lost && lane == 0) {
            tc_commit(bar(sh.drained));
            mbar_drain(bar(sh.drained), 0);
        }
        __syncwarp();
        tmem_dealloc(tmem);
    }
    if (lost) {
        if (tid == 0 && p.a.status) atomicOr(p.a.status, B200_DECODE_TIMEOUT);
        for (long long u = u_first; u < u_end;) {             // the join makes NaN of these
            const Part t = part_at(u);
            if (tid < kWideRows) p.part_ml[t.slot + tid] = make_float2(INFINITY, __int_as_float(0x7fffffff));
            u += t.n;
        }
    }
}

template <typename T, int D, int RING>
cudaError_t launch_ring(const AttnParams& p, size_t scan, cudaStream_t s) {
    const size_t smem = Wide<D, RING>::kBytes + sizeof(WideShared) + scan + 1024;
    const cudaError_t e = allow_smem<attn_wide_kernel<T, D, RING>>();
    if (e != cudaSuccess) return e;
    return launch_pdl(attn_wide_kernel<T, D, RING>, dim3((unsigned)p.grid), dim3(kThreads), smem, s, p);
}
template <typename T>
cudaError_t launch_typed(const AttnParams& p, cudaStream_t s) {
    const size_t scan = 8 * ((size_t)p.a.n_groups + 1);
    if (p.c.head_dim == 64) return launch_ring<T, 64, 8>(p, scan, s);
    // as many blocks as fit beside the scan's arrays
    if (Wide<128, 5>::kBytes + sizeof(WideShared) + scan + 1024 <= kSmemLimit) return launch_ring<T, 128, 5>(p, scan, s);
    return launch_ring<T, 128, 4>(p, scan, s);
}

}  // namespace

cudaError_t launch_attention_wide(const AttnParams& p, int dtype, cudaStream_t s) {
    return dtype == B200_LORA_F16 ? launch_typed<__half>(p, s) : launch_typed<__nv_bfloat16>(p, s);
}

}  // namespace b200lora
