// Decode attention over a paged cache, split along the keys: every warp takes a contiguous range of the work's units
// (see decode_common.cuh) and leaves the unnormalised sums, maximum and sum of exponentials of its part; a second
// kernel joins the parts of each query row.
//
// One pass over the keys with a running maximum m and sum l: with z = scale * q.k in powers of two,
//     m' = max(m, z_j)      l = l 2^(m - m') + sum 2^(z_j - m')      o = o 2^(m - m') + sum 2^(z_j - m') v_j
// A warp brings kKeys keys and values at a time into a ring of its own in shared memory by asynchronous copies (16
// bytes each, zeros in place of what lies behind the length or in a page that does not exist), so no barrier holds
// its neighbours up, and multiplies with mma.sync: decode reads every key for at most 16 query rows, some 16
// products a byte, so the copies bound it and not the multiplications.  The weights 2^(z - m) go into the second
// product as two 16-bit numbers (the value rounded, and what the rounding dropped), so nothing is lost against fp32.
//
// 32 requests of up to 2048 keys, 32 heads of 128: 112 us, 6.1 TB/s (677 MB; 93 % of what a copy reaches).  One
// request of 311 keys: 10 us, half of it latencies one after the other (lengths, page table, keys; parts, rows) and half the two launches.
#include <type_traits>

#include "attn_common.cuh"

namespace b200lora {

namespace {

constexpr int kKeys = kAttnKeys;
constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;

template <int D> struct Ring {
    static constexpr int kHalf = kKeys * D * 2;              // bytes of a stage's keys, or of its values
    static constexpr int kStage = 2 * kHalf;
    static constexpr int kStages = D == 128 ? 3 : 6;
    static constexpr int kBytes = kWarps * kStages * kStage;
};

__device__ __forceinline__ void ldsm4(unsigned addr, unsigned (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(unsigned addr, unsigned (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

template <int D>
__device__ __forceinline__ unsigned chunk_addr(unsigned base, int row, int chunk) {
    return base + row * (D * 2) + ((chunk ^ (row & 7)) << 4);
}

// The pages of the next kKeys keys of a page-table row: lane l holds key l % 16's.
struct PageWalk {
    const int* row;
    int keys;
};
__device__ __forceinline__ int page_at(const AttnParams& p, const PageWalk& w, int key0, int lane) {
    const int key = key0 + (lane & (kKeys - 1));
    return key < w.keys ? w.row[key >> p.page_shift] : kNoPage;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) attn_split_kernel(const __grid_constant__ AttnParams p) {
    extern __shared__ __align__(128) unsigned char smem[];
    using R = Ring<D>;
    int* su = reinterpret_cast<int*>(smem + R::kBytes);      // units before each entity
    int* st = su + p.a.n_groups + p.a.n_requests + 1;        // tiles before each group
    __shared__ unsigned long long warp_sum[kWarps];
    __shared__ int key_mask[kWarps][R::kStages];
    __shared__ int bad_all;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // The predecessor may be the wide kernel, which leaves alone what this one reads, but what came before that is only sure to be
    // seen by a grid that has waited itself.
    pdl_wait_prior();
    if (tid == 0) { pdl_launch_dependents(); bad_all = 0; }
    __syncthreads();
    int ignored = 0;
    // units before each entity, row tiles before each group; written out once for the join
    const int n_ent = p.a.n_groups + p.a.n_requests;
    const bool groups = scan_units<kThreads>(n_ent, p.a.n_groups, su, st, warp_sum, &bad_all, [&](int e, bool usable, int& bad) {
        const Entity t = split_entity(p, e, usable, bad);
        return ((unsigned long long)(e < p.a.n_groups ? t.tiles : 0) << 32) | (unsigned)(t.tiles * t.chunks);
    });
    if (blockIdx.x == 0) {
        for (int i = tid; i <= n_ent; i += kThreads) p.units[i] = su[i];
        for (int i = tid; i <= p.a.n_groups; i += kThreads) p.tiles[i] = groups ? st[i] : -1;
        if (tid == 0 && bad_all && p.a.status) atomicOr(p.a.status, bad_all);
    }

    const int n_kv = p.c.n_kv_heads;
    const long long total = (long long)su[n_ent] * n_kv;
    const int workers = (int)min((long long)gridDim.x * kWarps, total);
    const int worker = warp * gridDim.x + blockIdx.x;        // neighbours in the work on different SMs
    if (worker >= workers) return;
    long long u = unit_of_worker(total, worker, workers);
    const long long u_end = unit_of_worker(total, worker + 1, workers);
    const unsigned ring = smem_u32(smem) + warp * R::kStages * R::kStage;
    const int g4 = lane >> 2, t4 = lane & 3;

    while (u < u_end) {
        // ---- the item of unit u
        const int uh = (int)quotient(u, n_kv);
        const int e = entity_at(su, n_ent, uh);
        const Entity t = split_entity(p, e, groups, ignored);
        long long r = u - (long long)n_kv * su[e];
        const int per_head = t.tiles * t.chunks;
        const int h = (int)quotient(r, per_head);
        int rest = (int)(r - (long long)h * per_head);
        const int tile = rest / t.chunks, chunk0 = rest - tile * t.chunks;
        const int n = (int)min((long long)(t.chunks - chunk0), u_end - u);
        const bool group = e < p.a.n_groups;
        const int row0 = tile * kAttnRows, rows = min(kAttnRows, t.rows - row0);
        PageWalk walk;
        walk.row = group ? p.a.prefix_table + (long long)e * p.a.prefix_table_row
                         : p.a.table + (long long)(e - p.a.n_groups) * p.a.table_row;
        walk.keys = t.keys;

        // ---- query rows as A operands: row g4 and g4 + 8
        unsigned qa[D / 16][4];
        {
            const T* q0 = nullptr;
            const T* q1 = nullptr;
            const int ra = row0 + g4, rb = ra + 8;
            const int request_a = request_of_row(p, ra), request_b = request_of_row(p, rb);
            if (g4 < rows) q0 = static_cast<const T*>(p.a.q) + (long long)(t.first + request_a) * p.a.q_row + (long long)(h * p.per + ra - request_a * p.per) * p.a.q_head;
            if (g4 + 8 < rows) q1 = static_cast<const T*>(p.a.q) + (long long)(t.first + request_b) * p.a.q_row + (long long)(h * p.per + rb - request_b * p.per) * p.a.q_head;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                const int c = k * 16 + t4 * 2;
                qa[k][0] = q0 ? *reinterpret_cast<const unsigned*>(q0 + c) : 0u;
                qa[k][1] = q1 ? *reinterpret_cast<const unsigned*>(q1 + c) : 0u;
                qa[k][2] = q0 ? *reinterpret_cast<const unsigned*>(q0 + c + 8) : 0u;
                qa[k][3] = q1 ? *reinterpret_cast<const unsigned*>(q1 + c + 8) : 0u;
            }
        }
        float o[D / 8][4];
#pragma unroll
        for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

        // ---- keys: stage s of the ring holds step s, s + kStages, ...
        int page = page_at(p, walk, chunk0 * kKeys, lane);
        auto issue = [&](int step) {
            const int s = step % R::kStages;
            if (step < n) {
                const int key0 = (chunk0 + step) * kKeys;
                const bool fine = page >= 0 && page < p.c.n_pages;
                if (!fine && key0 + (lane & (kKeys - 1)) < walk.keys && p.a.status) atomicOr(p.a.status, B200_DECODE_BAD_PAGE);
                const long long off = fine ? (long long)page * p.c.page_stride +
                                                 (long long)((key0 + (lane & 15)) & ((1 << p.page_shift) - 1)) * p.c.token_stride
                                           : -1;
                const unsigned mask = __ballot_sync(0xffffffffu, fine) & 0xffffu;
                if (lane == 0) key_mask[warp][s] = (int)mask;
                if (step + 1 < n) page = page_at(p, walk, key0 + kKeys, lane);
                constexpr int kPerRow = D / 8, kRowsAt = 32 / kPerRow;
                const unsigned kdst = ring + s * R::kStage, vdst = kdst + R::kHalf;
                const T* kb = static_cast<const T*>(p.c.k) + (long long)h * p.c.head_stride;
                const T* vb = static_cast<const T*>(p.c.v) + (long long)h * p.c.head_stride;
#pragma unroll
                for (int i = 0; i < kKeys / kRowsAt; ++i) {
                    const int row = i * kRowsAt + lane / kPerRow, chunk = lane % kPerRow;
                    const long long ro = __shfl_sync(0xffffffffu, off, row);
                    const long long at = ro < 0 ? 0 : ro + chunk * 8;
                    cp_async16(chunk_addr<D>(kdst, row, chunk), kb + at, ro >= 0);
                    cp_async16(chunk_addr<D>(vdst, row, chunk), vb + at, ro >= 0);
                }
            }
            cp_commit();
        };
#pragma unroll
        for (int i = 0; i < R::kStages - 1; ++i) issue(i);
        for (int step = 0; step < n; ++step) {
            issue(step + R::kStages - 1);
            cp_wait<R::kStages - 1>();
            __syncwarp();
            const int s = step % R::kStages;
            const unsigned ks = ring + s * R::kStage, vs = ks + R::kHalf;
            const unsigned mask = (unsigned)key_mask[warp][s];
            float z[2][4] = {};
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                unsigned b[4];
                ldsm4(chunk_addr<D>(ks, (lane & 7) + ((lane >> 4) << 3), k * 2 + ((lane >> 3) & 1)), b);
                Mma<T>::run(z[0], qa[k][0], qa[k][1], qa[k][2], qa[k][3], b[0], b[1]);
                Mma<T>::run(z[1], qa[k][0], qa[k][1], qa[k][2], qa[k][3], b[2], b[3]);
            }
            float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const bool there = mask >> (i * 8 + t4 * 2 + j) & 1u;
                    z[i][j] = there ? z[i][j] * p.scale_log2 : -INFINITY;
                    z[i][2 + j] = there ? z[i][2 + j] * p.scale_log2 : -INFINITY;
                    x0 = fmaxf(x0, z[i][j]);
                    x1 = fmaxf(x1, z[i][2 + j]);
                }
            x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
            x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
            const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
            const float r0 = n0 == -INFINITY ? 0.f : n0, r1 = n1 == -INFINITY ? 0.f : n1;   // nothing yet: every weight is 0
            const float a0 = exp2f(m0 - r0), a1 = exp2f(m1 - r1);
            m0 = n0; m1 = n1;
            l0 *= a0; l1 *= a1;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    z[i][j] = exp2f(z[i][j] - r0);
                    z[i][2 + j] = exp2f(z[i][2 + j] - r1);
                    l0 += z[i][j];
                    l1 += z[i][2 + j];
                }
#pragma unroll
            for (int i = 0; i < D / 8; ++i) { o[i][0] *= a0; o[i][1] *= a0; o[i][2] *= a1; o[i][3] *= a1; }
            unsigned ph[4], pl[4];
            ph[0] = hl_pack<T>(z[0][0], z[0][1], false); pl[0] = hl_pack<T>(z[0][0], z[0][1], true);
            ph[1] = hl_pack<T>(z[0][2], z[0][3], false); pl[1] = hl_pack<T>(z[0][2], z[0][3], true);
            ph[2] = hl_pack<T>(z[1][0], z[1][1], false); pl[2] = hl_pack<T>(z[1][0], z[1][1], true);
            ph[3] = hl_pack<T>(z[1][2], z[1][3], false); pl[3] = hl_pack<T>(z[1][2], z[1][3], true);
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                unsigned b[4];
                ldsm4t(chunk_addr<D>(vs, (lane & 7) + ((lane >> 3) & 1) * 8, i * 2 + (lane >> 4)), b);
                Mma<T>::run(o[2 * i], ph[0], ph[1], ph[2], ph[3], b[0], b[1]);
                Mma<T>::run(o[2 * i + 1], ph[0], ph[1], ph[2], ph[3], b[2], b[3]);
                Mma<T>::run(o[2 * i], pl[0], pl[1], pl[2], pl[3], b[0], b[1]);
                Mma<T>::run(o[2 * i + 1], pl[0], pl[1], pl[2], pl[3], b[2], b[3]);
            }
            __syncwarp();                                      // the stage may be filled again
        }
        cp_wait<0>();

        // ---- the item's part of this worker
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1); l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1); l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
        const size_t slot_row = group
            ? ((size_t)n_kv * st[e] + (size_t)h * t.tiles + tile + worker) * kAttnRows
            : attn_group_rows(p) + (((size_t)(e - p.a.n_groups) * n_kv + h) * p.req_tiles + tile + worker) * p.req_rows;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int row = g4 + 8 * half;
            if (row >= rows) continue;
            float* dst = p.part + (slot_row + row) * D;
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
                *reinterpret_cast<float2*>(dst + i * 8 + t4 * 2) = half ? make_float2(o[i][2], o[i][3]) : make_float2(o[i][0], o[i][1]);
            if (t4 == 0) p.part_ml[slot_row + row] = half ? make_float2(m1, l1) : make_float2(m0, l0);
        }
        __syncwarp();
        u += n;
    }
}

constexpr int kJoin = 4;                          // parts whose rows are asked for together
// PER warps of a block per query row: the row's parts of its group's item and of its own item, weighted by 2^(m_i - max m).
constexpr int kJoinWarps = 8;
template <typename T, int D, int PER>
__global__ void __launch_bounds__(kJoinWarps * 32) attn_join_kernel(const __grid_constant__ AttnParams p) {
    constexpr int V = D / 32;
    __shared__ float all_acc[PER > 1 ? kJoinWarps : 1][D];
    __shared__ float2 all_ml[PER > 1 ? kJoinWarps : 1];
    pdl_wait_prior();
    if (threadIdx.x == 0) pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, mine = warp % PER;
    const long long n_rows = (long long)p.a.n_requests * p.a.n_heads, row_all = (long long)blockIdx.x * (kJoinWarps / PER) + warp / PER;
    const bool there = row_all < n_rows;
    if (PER == 1 && !there) return;
    float acc[V], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = 0.f;
    if (there) {
        const int b = (int)quotient(row_all, p.a.n_heads), hq = (int)(row_all - (long long)b * p.a.n_heads);
        const int h = hq / p.per, i = hq - h * p.per, n_kv = p.c.n_kv_heads, n_g = p.a.n_groups;
        const int n_ent = n_g + p.a.n_requests;
        const long long total = (long long)p.units[n_ent] * n_kv;
        const int workers = (int)min((long long)p.grid * kWarps, total);

        // The row's parts: those of its group's item (a wide tile of one stream's rows has a second part for each), then of its own.  Part
        // i of a run lies at row first + i * pitch.
        struct Run { size_t first; int pitch, n; } run[3] = {{0, 0, 0}, {0, 0, 0}, {0, 0, 0}};
        if (n_g > 0 && p.tiles[0] >= 0) {                          // starts ascend
            int lo = -1, hi = n_g;                                 // last group that starts at or before b
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (p.a.group_starts[mid] <= b) lo = mid; else hi = mid;
            }
            if (lo >= 0 && b < p.a.group_starts[lo + 1]) {
                const int r = (b - p.a.group_starts[lo]) * p.per + i, n_rows = (p.a.group_starts[lo + 1] - p.a.group_starts[lo]) * p.per;
                const bool wide = n_rows > kWideFrom;
                const int* units = wide ? p.wide_units : p.units;
                const int* before = wide ? p.wide_tile : p.tiles;
                const int tiles = before[lo + 1] - before[lo], all = units[lo + 1] - units[lo], tile = r / (wide ? kWideRows : kAttnRows);
                if (all > 0) {
                    const int chunks = all / tiles;
                    const long long u0 = (long long)n_kv * units[lo] + (long long)h * all + (long long)tile * chunks;
                    const size_t item = (size_t)n_kv * before[lo] + (size_t)h * tiles + tile;
                    const long long sum = wide ? (long long)p.wide_units[n_g] * n_kv : total;
                    const int w = wide ? (int)min((long long)p.grid, sum) : workers;
                    const int w0 = worker_of_unit(sum, u0, w), n = worker_of_unit(sum, u0 + chunks - 1, w) - w0 + 1;
                    if (!wide) run[0] = {(item + w0) * kAttnRows + (r - tile * kAttnRows), kAttnRows, n};
                    else {
                        run[0] = {attn_group_rows(p) + attn_request_rows(p) + (item + w0) * kWideRows + (r - tile * kWideRows), kWideRows, n};
                        if (n_rows - tile * kWideRows <= kWideRows / 2) run[1] = {run[0].first + kWideRows / 2, kWideRows, n};
                    }
                }
            }
        }
        const int e = n_g + b, all = p.units[e + 1] - p.units[e];
        if (all > 0) {
            const int chunks = all / p.req_tiles, tile = i / kAttnRows;
            const long long u0 = (long long)n_kv * p.units[e] + (long long)h * all + (long long)tile * chunks;
            const size_t item = ((size_t)b * n_kv + h) * p.req_tiles + tile;
            const int w0 = worker_of_unit(total, u0, workers);
            run[2] = {attn_group_rows(p) + (item + w0) * p.req_rows + (i - tile * kAttnRows), p.req_rows, worker_of_unit(total, u0 + chunks - 1, workers) - w0 + 1};
        }
        auto part_at = [&](int k) {
            if (k < run[0].n) return run[0].first + (size_t)k * run[0].pitch;
            k -= run[0].n;
            if (k < run[1].n) return run[1].first + (size_t)k * run[1].pitch;
            return run[2].first + (size_t)(k - run[1].n) * run[2].pitch;
        };
        const int all_parts = run[0].n + run[1].n + run[2].n, parts = (all_parts - mine + PER - 1) / PER;   // every PERth is this warp's
        for (int base = 0; base < parts; base += 32) {
            // a part a lane: maxima and sums
            const int n = min(32, parts - base);
            const size_t at = part_at((base + min(lane, n - 1)) * PER + mine);
            const float2 ml = lane < n ? __ldcg(p.part_ml + at) : make_float2(-INFINITY, 0.f);
            float top = ml.x;
#pragma unroll
            for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float to = fmaxf(m, top), ref = to == -INFINITY ? 0.f : to;
            const float old = exp2f(m - ref), w = exp2f(ml.x - ref);
            m = to;
            float sum = w * ml.y;
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            l = l * old + sum;
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] *= old;
            for (int j = 0; j < n; j += kJoin) {
                // the rows of kJoin parts are asked for together; those of a part without keys may be anything
                float f[kJoin][V];
#pragma unroll
                for (int k = 0; k < kJoin; ++k) {
                    const float* src = p.part + __shfl_sync(0xffffffffu, at, min(j + k, n - 1)) * D + lane * V;
                    if constexpr (V == 4) {
                        const float4 g = __ldcg(reinterpret_cast<const float4*>(src));
                        f[k][0] = g.x; f[k][1] = g.y; f[k][2] = g.z; f[k][3] = g.w;
                    } else {
                        const float2 g = __ldcg(reinterpret_cast<const float2*>(src));
                        f[k][0] = g.x; f[k][1] = g.y;
                    }
                }
#pragma unroll
                for (int k = 0; k < kJoin; ++k) {
                    const float wk = __shfl_sync(0xffffffffu, w, min(j + k, 31));
                    if (j + k < n && wk != 0.f)
#pragma unroll
                        for (int c = 0; c < V; ++c) acc[c] += wk * f[k][c];
                }
            }
        }
    }
    if constexpr (PER > 1) {
        // the warps of a row
#pragma unroll
        for (int k = 0; k < V; ++k) all_acc[warp][k * 32 + lane] = acc[k];
        if (lane == 0) all_ml[warp] = make_float2(m, l);
        __syncthreads();
        if (mine != 0 || !there) return;
        float top = m;
#pragma unroll
        for (int w = 1; w < PER; ++w) top = fmaxf(top, all_ml[warp + w].x);
        const float ref = top == -INFINITY ? 0.f : top;
        m = top;
        l = 0.f;
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] = 0.f;
#pragma unroll
        for (int w = 0; w < PER; ++w) {
            const float2 ml = all_ml[warp + w];
            const float f = exp2f(ml.x - ref);
            l += f * ml.y;
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] += f * all_acc[warp + w][k * 32 + lane];
        }
    }
    const long long b = quotient(row_all, p.a.n_heads), hq = row_all - b * p.a.n_heads;
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;  // no key: zeros; NaN stays NaN
    T* out = static_cast<T*>(p.a.out) + b * p.a.out_row + hq * p.a.out_head + lane * V;
    if constexpr (V == 4) {
        uint2 u;
        u.x = Cvt<T>::pack2(acc[0] * inv, acc[1] * inv);
        u.y = Cvt<T>::pack2(acc[2] * inv, acc[3] * inv);
        *reinterpret_cast<uint2*>(out) = u;
    } else *reinterpret_cast<unsigned*>(out) = Cvt<T>::pack2(acc[0] * inv, acc[1] * inv);
    if (p.a.lse && lane == 0) p.a.lse[row_all] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

template <typename T, int D>
cudaError_t launch_typed(const AttnParams& p0, int n_sm, cudaStream_t s) {
    AttnParams p = p0;
    const int grid = n_sm < kAttnMaxWorkers / kWarps ? n_sm : kAttnMaxWorkers / kWarps;
    p.grid = grid;
    const size_t smem = Ring<D>::kBytes + 4 * ((size_t)2 * p.a.n_groups + p.a.n_requests + 2);
    cudaError_t e = cudaSuccess;
    if (p.wide_tiles) {
        e = launch_attention_wide(p, std::is_same_v<T, __half> ? B200_LORA_F16 : B200_LORA_BF16, s);
        if (e != cudaSuccess) return e;
    }
    e = allow_smem<attn_split_kernel<T, D>>();
    if (e != cudaSuccess) return e;
    e = launch_pdl(attn_split_kernel<T, D>, grid, kThreads, smem, s, p);
    if (e != cudaSuccess) return e;
    // Eight warps for a row where the rows are few: there its parts are many (32 rows of 311 keys: 11.7 us with one warp, 10.1 us; 4096
    // rows of 8704 keys: 69 us with one, 89 us with eight).
    const unsigned rows = (unsigned)p.a.n_requests * p.a.n_heads;
    if (rows <= (unsigned)n_sm * 2) return launch_pdl(attn_join_kernel<T, D, kJoinWarps>, rows, kJoinWarps * 32, 0, s, p);
    return launch_pdl(attn_join_kernel<T, D, 1>, (rows + kJoinWarps - 1) / kJoinWarps, kJoinWarps * 32, 0, s, p);
}

}  // namespace

cudaError_t launch_attention(const AttnParams& p, int dtype, int n_sm, cudaStream_t s) {
    if (dtype == B200_LORA_F16) return p.c.head_dim == 128 ? launch_typed<__half, 128>(p, n_sm, s) : launch_typed<__half, 64>(p, n_sm, s);
    return p.c.head_dim == 128 ? launch_typed<__nv_bfloat16, 128>(p, n_sm, s) : launch_typed<__nv_bfloat16, 64>(p, n_sm, s);
}

}  // namespace b200lora
