// What the attention kernels share: entities, their units, the split of the units over workers (sm_100a).
#pragma once

#include "decode_common.cuh"
#include "lora_pipe.cuh"

namespace b200lora {

namespace {

// a / b of numbers that are not negative and seldom have more than 32 bits: a division of 64-bit ones takes some 400 cycles
__device__ __forceinline__ long long quotient(long long a, long long b) {
    return ((a | b) >> 32) == 0 ? (long long)((unsigned)a / (unsigned)b) : a / b;
}
// Request of a group's row: row / per by multiplication, exact as long as row * per < 2^32 (rows <= 4096 * per, per <= 1024)
__device__ __forceinline__ int request_of_row(const AttnParams& p, int row) { return p.per == 1 ? row : (int)__umulhi((unsigned)row, p.per_inverse); }

struct Entity { int rows, tiles, chunks, keys, first; };     // first: request of the first row

__device__ __forceinline__ int clamped_keys(const AttnParams& p, int n, int pages, int& bad) {
    const int most = pages << p.page_shift;                   // fits: checked on the host
    if (n < 0 || n > most) bad |= B200_DECODE_BAD_LENGTH;
    return n < 0 ? 0 : n > most ? most : n;
}
// Group e, cut into tiles of TILE rows and chunks of KEYS keys.  `usable` false: the group starts cannot be used and no
// group has rows.  Groups of more than kWideFrom rows are the wide kernel's, the others the split kernel's.
template <int TILE, int KEYS, bool WIDE>
__device__ __forceinline__ Entity group_of(const AttnParams& p, int e, bool usable, int& bad) {
    Entity t;
    const int s0 = p.a.group_starts[e], s1 = p.a.group_starts[e + 1];
    const bool fine = s0 >= 0 && s1 >= s0 && s1 <= p.a.n_requests;
    if (!fine) bad |= B200_DECODE_BAD_GROUPS;
    t.first = s0;
    t.rows = fine && usable ? (s1 - s0) * p.per : 0;
    if ((t.rows > kWideFrom) != WIDE) t.rows = 0;
    t.tiles = (t.rows + TILE - 1) / TILE;
    t.keys = clamped_keys(p, p.a.prefix_lens[e], p.a.max_prefix_pages, bad);
    if (t.rows == 0) t.keys = 0;
    t.chunks = (t.keys + KEYS - 1) / KEYS;
    return t;
}

// Entity e of the split kernel: group e, or request e - n_groups
__device__ __forceinline__ Entity split_entity(const AttnParams& p, int e, bool usable, int& bad) {
    if (e < p.a.n_groups) return group_of<kAttnRows, kAttnKeys, false>(p, e, usable, bad);
    Entity t;
    t.first = e - p.a.n_groups;
    t.rows = p.per;
    t.tiles = p.req_tiles;
    t.keys = clamped_keys(p, p.a.lens[t.first], p.a.max_pages, bad);
    t.chunks = (t.keys + kAttnKeys - 1) / kAttnKeys;
    return t;
}

// Units before each entity (su[0..n]) and row tiles before each (st[0..n_tiles_of]); value(e, usable, bad) gives tiles << 32 | units
// of entity e.  Starts that descend somewhere leave every group out (returns whether groups can be used).
template <int THREADS, typename F>
__device__ __forceinline__ bool scan_units(int n, int n_groups, int* su, int* st, unsigned long long* warp_sum, int* bad_all, F value) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    bool usable = n_groups > 0;
    for (int attempt = 0; attempt < 2; ++attempt) {
        unsigned long long carry = 0;
        int bad = 0;
        for (int base = 0; base < n; base += THREADS) {
            const int e = base + tid;
            const unsigned long long v = e < n ? value(e, usable, bad) : 0ull;
            unsigned long long inc = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long up = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += up;
            }
            if (lane == 31) warp_sum[warp] = inc;
            __syncthreads();
            unsigned long long before = carry, all = 0;
#pragma unroll
            for (int w = 0; w < THREADS / 32; ++w) { if (w < warp) before += warp_sum[w]; all += warp_sum[w]; }
            if (e < n) {
                su[e] = (int)(unsigned)(before + inc - v);
                if (e < n_groups) st[e] = (int)((before + inc - v) >> 32);
            }
            carry += all;
            __syncthreads();
        }
        if (tid == 0) { su[n] = (int)(unsigned)carry; st[n_groups] = (int)(carry >> 32); }
        if (bad) atomicOr(bad_all, bad);
        __syncthreads();
        if (!usable || !(*bad_all & B200_DECODE_BAD_GROUPS)) break;
        usable = false;
    }
    return usable;
}

// last entity with su[e] <= uh
__device__ __forceinline__ int entity_at(const int* su, int n, int uh) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (su[mid] <= uh) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ long long unit_of_worker(long long total, int w, int workers) { return quotient(total * w, workers); }
__device__ __forceinline__ int worker_of_unit(long long total, long long u, int workers) {
    return (int)quotient((u + 1) * workers - 1, total);
}

// What stands for the page of a key behind the length: never one of the cache's, but a page table can hold the same number, so whether
// a key is there is asked of its index.
constexpr int kNoPage = -1;

__device__ __forceinline__ void cp_async16(unsigned dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

}  // namespace

}  // namespace b200lora
