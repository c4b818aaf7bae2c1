// Append: LoRA deltas added, q and k rotated by position, k and v to their slots of a paged cache, in one pass.
//
// A rotation by the angle a of a pair (x0, x1): (x0 cos a - x1 sin a, x1 cos a + x0 sin a).  Every element is read
// once and written once, so the bytes bound the kernel, or its launch when tokens are few.  A thread holds one unit
// (2 * VEC elements that rotate among themselves) of a head and keeps its cosines and sines while it goes through
// the token's heads: the tables are then read once per token and block, and no shuffle is needed.
#include "decode_common.cuh"

namespace b200lora {

namespace {

constexpr int kAppendThreads = 256;

struct AppendParams {
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

template <typename T, int VEC>
__device__ __forceinline__ void load(const T* p, float (&f)[VEC]) {
    if constexpr (VEC == 8) Cvt<T>::unpack8(*reinterpret_cast<const uint4*>(p), f);
    else f[0] = to_f<T>(*p);
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
    if (!f32) { load<T, VEC>(static_cast<const T*>(tab) + at, f); return; }
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
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const __grid_constant__ AppendParams p) {
    pdl_wait_prior();
    if (threadIdx.x == 0) pdl_launch_dependents();
    const b200_append& a = p.a;
    const int lane_head = threadIdx.x / p.units, unit = threadIdx.x - lane_head * p.units;
    const int sub = lane_head / p.heads_per_pass;
    const long long t = (long long)blockIdx.x * p.tokens_per_block + sub;
    if (sub >= p.tokens_per_block || t >= a.n_tokens) return;
    const long long slot = index_at(a.slots, a.slots_are_i64, t);
    if (slot < 0) return;
    const long long pos = index_at(a.positions, a.positions_are_i64, t);
    const long long page = slot / p.c.page_size;
    const int bad = (page >= p.c.n_pages ? B200_DECODE_BAD_SLOT : 0) | (pos < 0 || pos >= a.n_positions ? B200_DECODE_BAD_POSITION : 0);
    if (bad) {
        if (a.status && unit == 0) atomicOr(a.status, bad);
        return;
    }
    const long long place = page * p.c.page_stride + (slot - page * p.c.page_size) * p.c.token_stride;
    const int n_q = a.n_heads, n_kv = p.c.n_kv_heads, n_all = n_q + 2 * n_kv;
    const bool turned = unit * 2 * VEC < a.rotary_dim;
    const bool halves = turned && !a.interleaved;
    const int lo = halves ? unit * VEC : unit * 2 * VEC, hi = halves ? lo + a.rotary_dim / 2 : lo + VEC;
    const int vlo = unit * 2 * VEC, vhi = vlo + VEC;      // of v, which is not turned
    float cs[VEC], sn[VEC];
    if (turned) {
        load_table<T, VEC>(a.cos, a.tables_are_f32, pos * a.table_row + unit * VEC, cs);
        load_table<T, VEC>(a.sin, a.tables_are_f32, pos * a.table_row + unit * VEC, sn);
    }
    for (int h = (int)blockIdx.y * p.heads_per_pass + lane_head - sub * p.heads_per_pass; h < n_all; h += gridDim.y * p.heads_per_pass) {
        const bool is_q = h < n_q, is_v = h >= n_q + n_kv;
        const int hh = is_q ? h : is_v ? h - n_q - n_kv : h - n_q;
        const T* x = static_cast<const T*>(is_q ? a.q : is_v ? a.v : a.k) +
                     t * (is_q ? a.q_row : is_v ? a.v_row : a.k_row) + hh * (is_q ? a.q_head : is_v ? a.v_head : a.k_head);
        const T* dx = static_cast<const T*>(is_q ? a.dq : is_v ? a.dv : a.dk);
        T* y = is_q ? static_cast<T*>(a.q_out) + t * a.q_out_row + hh * a.q_out_head
                    : static_cast<T*>(is_v ? p.c.v : p.c.k) + place + hh * p.c.head_stride;
        const int at0 = is_v ? vlo : lo, at1 = is_v ? vhi : hi;
        float f0[VEC], f1[VEC];
        load<T, VEC>(x + at0, f0);
        load<T, VEC>(x + at1, f1);
        if (dx) {
            dx += t * (is_q ? a.dq_row : is_v ? a.dv_row : a.dk_row) + hh * (is_q ? a.dq_head : is_v ? a.dv_head : a.dk_head);
            float d0[VEC], d1[VEC];
            load<T, VEC>(dx + at0, d0);
            load<T, VEC>(dx + at1, d1);
#pragma unroll
            for (int i = 0; i < VEC; ++i) { f0[i] += d0[i]; f1[i] += d1[i]; }
        }
        if (turned && !is_v) {
            auto turn = [](float& x0, float& x1, float c, float s) {
                const float y0 = x0 * c - x1 * s, y1 = x1 * c + x0 * s;
                x0 = y0; x1 = y1;
            };
            if (a.interleaved) {
                if constexpr (VEC == 1) turn(f0[0], f1[0], cs[0], sn[0]);
                else {
#pragma unroll
                    for (int i = 0; i < VEC / 2; ++i) {
                        turn(f0[2 * i], f0[2 * i + 1], cs[i], sn[i]);
                        turn(f1[2 * i], f1[2 * i + 1], cs[VEC / 2 + i], sn[VEC / 2 + i]);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) turn(f0[i], f1[i], cs[i], sn[i]);
            }
        }
        store<T, VEC>(y + at0, f0);
        store<T, VEC>(y + at1, f1);
    }
}

}  // namespace

cudaError_t launch_kv_append(const b200_append& a, const b200_kv_cache& c, int dtype, bool vectors, cudaStream_t s) {
    AppendParams p;
    p.a = a; p.c = c;
    p.units = c.head_dim / (vectors ? 16 : 2);
    const int lanes = kAppendThreads / p.units, heads = a.n_heads + 2 * c.n_kv_heads;
    p.heads_per_pass = lanes < heads ? lanes : heads;
    p.tokens_per_block = lanes / p.heads_per_pass;
    const unsigned blocks = (unsigned)((a.n_tokens + (long long)p.tokens_per_block - 1) / p.tokens_per_block);
    // few tokens: one pass per block, so that all heads move at once
    const int passes = (heads + p.heads_per_pass - 1) / p.heads_per_pass;
    const dim3 grid(blocks, (unsigned)passes);
    if (dtype == B200_LORA_F16)
        return launch_pdl(vectors ? kv_append_kernel<__half, 8> : kv_append_kernel<__half, 1>, grid, kAppendThreads, 0, s, p);
    return launch_pdl(vectors ? kv_append_kernel<__nv_bfloat16, 8> : kv_append_kernel<__nv_bfloat16, 1>, grid, kAppendThreads, 0, s, p);
}

}  // namespace b200lora
