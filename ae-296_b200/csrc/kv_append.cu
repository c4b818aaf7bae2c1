// Append: LoRA deltas added, q and k rotated by position, k and v to their slots of a paged cache, in one pass.
//
// A rotation by the angle a of a pair (x0, x1): (x0 cos a - x1 sin a, x1 cos a + x0 sin a).  Every element is read
// once and written once, so the bytes bound the kernel, or its launch when tokens are few.  A thread holds one unit
// (2 * VEC elements that rotate among themselves) of a head and keeps its cosines and sines while it goes through
// the token's heads: the tables are then read once per token and block, and no shuffle is needed.
//
// 8191 tokens of 40+40+40 heads of 128: 92 us, 5.3 TB/s of reading and writing (74 us at a copy's 6.55 TB/s).  What is read is asked
// for before the token's slot is known, which brought 160 us down to 92 us together with four blocks an SM (with five
// registers spill).  256 tokens of 64+8+8 heads with deltas: 4.7 us; one token: 4.2 us, of which the launch is nearly all.
#include "decode_common.cuh"

namespace b200lora {

namespace {

constexpr int kAppendThreads = 256;
constexpr int kBlocksPerSm = 16;

struct Side { const void *x, *dx; void* y; long long x_row, x_head, dx_row, dx_head, y_head; };     // q, k or v
struct AppendParams {
    Side side[3];
    b200_append a;
    b200_kv_cache c;
    int units;             // of a head
    int heads_per_pass;    // heads of a token that a block takes at a time
    int tokens_per_block;
};

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// VEC elements as they are in memory
template <typename T, int VEC> struct Raw { uint4 v; };
template <typename T> struct Raw<T, 1> { T v; };
template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> fetch(const T* p) { return *reinterpret_cast<const Raw<T, VEC>*>(p); }
template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Raw<T, VEC>& r, float (&f)[VEC]) {
    if constexpr (VEC == 8) Cvt<T>::unpack8(r.v, f);
    else f[0] = to_f<T>(r.v);
}
template <typename T, int VEC>
__device__ __forceinline__ void store(T* p, const float (&f)[VEC]) {
    if constexpr (VEC == 8) {
        uint4 u;
        u.x = Cvt<T>::pack2(f[0], f[1]); u.y = Cvt<T>::pack2(f[2], f[3]);
        u.z = Cvt<T>::pack2(f[4], f[5]); u.w = Cvt<T>::pack2(f[6], f[7]);
        *reinterpret_cast<uint4*>(p) = u;
    } else *p = from_f<T>(f[0]);
}
template <typename T, int VEC>
__device__ __forceinline__ void load_table(const void* tab, int f32, long long at, float (&f)[VEC]) {
    if (!f32) { unpack<T, VEC>(fetch<T, VEC>(static_cast<const T*>(tab) + at), f); return; }
    const float* p = static_cast<const float*>(tab) + at;
    if constexpr (VEC == 8) {
        const float4 lo = reinterpret_cast<const float4*>(p)[0], hi = reinterpret_cast<const float4*>(p)[1];
        f[0] = lo.x; f[1] = lo.y; f[2] = lo.z; f[3] = lo.w; f[4] = hi.x; f[5] = hi.y; f[6] = hi.z; f[7] = hi.w;
    } else f[0] = *p;
}
__device__ __forceinline__ long long index_at(const void* p, int i64, long long t) {
    return i64 ? static_cast<const long long*>(p)[t] : (long long)static_cast<const int*>(p)[t];
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kAppendThreads, 4) kv_append_kernel(const __grid_constant__ AppendParams p) {
    pdl_wait_prior();
    if (threadIdx.x == 0) pdl_launch_dependents();
    const b200_append& a = p.a;
    const int lane_head = threadIdx.x / p.units, unit = threadIdx.x - lane_head * p.units;
    const int sub = lane_head / p.heads_per_pass;
    const long long t = (long long)blockIdx.x * p.tokens_per_block + sub;
    if (sub >= p.tokens_per_block || t >= a.n_tokens) return;
    const long long slot = index_at(a.slots, a.slots_are_i64, t);
    const long long pos = index_at(a.positions, a.positions_are_i64, t);
    const int n_q = a.n_heads, n_kv = p.c.n_kv_heads, n_all = n_q + 2 * n_kv;
    const bool turned = unit * 2 * VEC < a.rotary_dim;
    const bool halves = turned && !a.interleaved;
    const int lo = halves ? unit * VEC : unit * 2 * VEC, hi = halves ? lo + a.rotary_dim / 2 : lo + VEC;
    const int vlo = unit * 2 * VEC, vhi = vlo + VEC;      // of v, which is not turned
    const int step = gridDim.y * p.heads_per_pass;
    Raw<T, VEC> x0, x1, d0, d1;
    int which = 0, at0 = 0, at1 = 0;
    long long head = 0;
    auto ask = [&](int h) {
        which = h < n_q ? 0 : h < n_q + n_kv ? 1 : 2;
        head = h - (which == 0 ? 0 : which == 1 ? n_q : n_q + n_kv);
        at0 = which == 2 ? vlo : lo;
        at1 = which == 2 ? vhi : hi;
        const Side& s = p.side[which];
        const T* from = static_cast<const T*>(s.x) + t * s.x_row + head * s.x_head;
        x0 = fetch<T, VEC>(from + at0);
        x1 = fetch<T, VEC>(from + at1);
        if (s.dx) {
            const T* more = static_cast<const T*>(s.dx) + t * s.dx_row + head * s.dx_head;
            d0 = fetch<T, VEC>(more + at0);
            d1 = fetch<T, VEC>(more + at1);
        }
    };
    int h = (int)blockIdx.y * p.heads_per_pass + lane_head - sub * p.heads_per_pass;
    if (h >= n_all) return;
    ask(h);                                               // (also for a row that is left out: q, k and v have it)
    if (slot < 0) return;
    const long long page = slot / p.c.page_size;
    const int bad = (page >= p.c.n_pages ? B200_DECODE_BAD_SLOT : 0) | (pos < 0 || pos >= a.n_positions ? B200_DECODE_BAD_POSITION : 0);
    if (bad) {
        if (a.status && unit == 0) atomicOr(a.status, bad);
        return;
    }
    const long long place = page * p.c.page_stride + (slot - page * p.c.page_size) * p.c.token_stride;
    float cs[VEC], sn[VEC];
    if (turned) {
        load_table<T, VEC>(a.cos, a.tables_are_f32, pos * a.table_row + unit * VEC, cs);
        load_table<T, VEC>(a.sin, a.tables_are_f32, pos * a.table_row + unit * VEC, sn);
    }
    while (true) {
        const Side& s = p.side[which];
        float f0[VEC], f1[VEC];
        unpack<T, VEC>(x0, f0);
        unpack<T, VEC>(x1, f1);
        if (s.dx) {
            float e0[VEC], e1[VEC];
            unpack<T, VEC>(d0, e0);
            unpack<T, VEC>(d1, e1);
#pragma unroll
            for (int k = 0; k < VEC; ++k) { f0[k] += e0[k]; f1[k] += e1[k]; }
        }
        if (turned && which < 2) {
            auto turn = [](float& u, float& v, float c, float s) {
                const float y0 = u * c - v * s, y1 = v * c + u * s;
                u = y0; v = y1;
            };
            if (a.interleaved) {
                if constexpr (VEC == 1) turn(f0[0], f1[0], cs[0], sn[0]);
                else {
#pragma unroll
                    for (int k = 0; k < VEC / 2; ++k) {
                        turn(f0[2 * k], f0[2 * k + 1], cs[k], sn[k]);
                        turn(f1[2 * k], f1[2 * k + 1], cs[VEC / 2 + k], sn[VEC / 2 + k]);
                    }
                }
            } else {
#pragma unroll
                for (int k = 0; k < VEC; ++k) turn(f0[k], f1[k], cs[k], sn[k]);
            }
        }
        T* y = static_cast<T*>(s.y) + (which == 0 ? t * a.q_out_row : place) + head * s.y_head;
        store<T, VEC>(y + at0, f0);
        store<T, VEC>(y + at1, f1);
        h += step;
        if (h >= n_all) return;
        ask(h);
    }
}

}  // namespace

cudaError_t launch_kv_append(const b200_append& a, const b200_kv_cache& c, int dtype, bool vectors, int n_sm, cudaStream_t s) {
    AppendParams p;
    p.a = a; p.c = c;
    p.side[0] = {a.q, a.dq, a.q_out, a.q_row, a.q_head, a.dq_row, a.dq_head, a.q_out_head};
    p.side[1] = {a.k, a.dk, c.k, a.k_row, a.k_head, a.dk_row, a.dk_head, c.head_stride};
    p.side[2] = {a.v, a.dv, c.v, a.v_row, a.v_head, a.dv_row, a.dv_head, c.head_stride};
    p.units = c.head_dim / (vectors ? 16 : 2);
    const int lanes = kAppendThreads / p.units, heads = a.n_heads + 2 * c.n_kv_heads;
    p.heads_per_pass = lanes < heads ? lanes : heads;
    p.tokens_per_block = lanes / p.heads_per_pass;
    const unsigned blocks = (unsigned)((a.n_tokens + (long long)p.tokens_per_block - 1) / p.tokens_per_block);
    // Few tokens: one pass per block, so that all heads move at once.  Many: a block keeps a token's sines and its address for as
    // many heads as leave about kBlocksPerSm blocks for every SM.
    const int passes = (heads + p.heads_per_pass - 1) / p.heads_per_pass;
    const unsigned want = (unsigned)(kBlocksPerSm * n_sm) / blocks + 1;
    const dim3 grid(blocks, want < (unsigned)passes ? want : (unsigned)passes);
    if (dtype == B200_LORA_F16)
        return launch_pdl(vectors ? kv_append_kernel<__half, 8> : kv_append_kernel<__half, 1>, grid, kAppendThreads, 0, s, p);
    return launch_pdl(vectors ? kv_append_kernel<__nv_bfloat16, 8> : kv_append_kernel<__nv_bfloat16, 1>, grid, kAppendThreads, 0, s, p);
}

}  // namespace b200lora
