// What the kernels of the products with 4-bit weights share (sm_100a).
#pragma once

#include <initializer_list>

#include "decode_common.cuh"
#include "tc_common.cuh"

namespace b200lora {

constexpr int kInt4MaxSplit = 8;              // blocks of a cluster that share a tile's columns

struct Int4Params {
    alignas(64) CUtensorMap codes, x;
    b200_int4 a;
    int y_f32, split, x_panels, early;       // early: a successor's blocks may come at once
};

namespace {

// Pairs of 16-bit numbers from the subnormal numbers that the bits of codes are: fma(c, o) = c / kInverse + o.
template <typename T> struct Codes;
template <> struct Codes<__half> {                            // c 2^-24 * 2^15, or 16 c 2^-24 * 2^11
    static constexpr float kInverse = 512.f;
    static __device__ __forceinline__ unsigned fma(unsigned v, unsigned o) {
        const unsigned up = 0x68007800u;
        const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&up), *reinterpret_cast<const __half2*>(&o));
        return *reinterpret_cast<const unsigned*>(&r);
    }
};
template <> struct Codes<__nv_bfloat16> {                     // c 2^-133 * 2^127, or 16 c 2^-133 * 2^123
    static constexpr float kInverse = 64.f;
    static __device__ __forceinline__ unsigned fma(unsigned v, unsigned o) {
        const unsigned up = 0x7d007f00u;
        const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&up), *reinterpret_cast<const __nv_bfloat162*>(&o));
        return *reinterpret_cast<const unsigned*>(&r);
    }
};
template <typename T> __device__ __forceinline__ float from_bits(unsigned short u);
template <> __device__ __forceinline__ float from_bits<__half>(unsigned short u) { return __half2float(__ushort_as_half(u)); }
template <> __device__ __forceinline__ float from_bits<__nv_bfloat16>(unsigned short u) { return __uint_as_float((unsigned)u << 16); }

__device__ __forceinline__ void prefetch_tensor(const void* map, int x, int y) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ float4 remote_f32x4(unsigned addr, unsigned rank) {
    float4 v;
    asm volatile("{ .reg .b32 r; mapa.shared::cluster.u32 r, %4, %5; ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [r]; }"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr), "r"(rank) : "memory");
    return v;
}
// Eight columns, in order, of a word of codes; o: what takes the zero point away (zero_offset).  Columns 2 i are the low four bits of
// byte i and become the low halves of the pairs; columns 2 i + 1 stay 16 times as large in the high ones, and the multiplier
// differs instead.  The zero bytes between are the sign, eight times, of a byte that is below 128.
template <typename T> __device__ __forceinline__ unsigned zero_offset(unsigned z) { return Codes<T>::fma(z * 0x00100001u, 0u) ^ 0x80008000u; }
template <unsigned SEL> __device__ __forceinline__ unsigned permute(unsigned a, unsigned b);
template <typename T> __device__ __forceinline__ void eight_columns(unsigned w, unsigned o, unsigned (&v)[4]) {
    const unsigned even = w & 0x0f0f0f0fu, odd = w & 0xf0f0f0f0u;
    v[0] = Codes<T>::fma(permute<0x8480>(even, odd), o);
    v[1] = Codes<T>::fma(permute<0x9591>(even, odd), o);
    v[2] = Codes<T>::fma(permute<0xa6a2>(even, odd), o);
    v[3] = Codes<T>::fma(permute<0xb7b3>(even, odd), o);
}
// bytes of (a, b) by the nibbles of SEL; 8 + i is the sign of byte i, eight times
template <unsigned SEL> __device__ __forceinline__ unsigned permute(unsigned a, unsigned b) {
    unsigned r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "n"(SEL));
    return r;
}
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
__device__ __forceinline__ void tensor_g2s_3d(unsigned dst, const void* map, int x, int y, int z, unsigned bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}

// Adds up the sums of a cluster's blocks (or of the only one), `add`, and stores y: red [TOKENS][PITCH] holds this block's sums of
// 128 rows and is read by the others; a thread takes four rows of a token.
template <typename T, int TOKENS, int PITCH, int THREADS>
__device__ __forceinline__ void finish_sums(const Int4Params& p, const float* red, int row0, int tok0, int part) {
    const b200_int4& a = p.a;
    constexpr int kQuads = kTcRows / 4;
    const int tid = threadIdx.x;
    if (p.split > 1) cluster_sync(); else __syncthreads();
    for (int e = part * THREADS + tid; e < TOKENS * kQuads; e += p.split * THREADS) {
        const int tok = e / kQuads, row = e % kQuads * 4, col = row0 + row;
        if (tok0 + tok >= a.n_tokens) break;                  // tokens ascend
        if (col >= a.n_out) continue;
        const long long to = (long long)(tok0 + tok) * a.y_row + col, from = (long long)(tok0 + tok) * a.add_row + col;
        float f[4], g[4] = {0.f, 0.f, 0.f, 0.f};
        if (a.add)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (col + i < a.n_out) g[i] = p.y_f32 ? static_cast<const float*>(a.add)[from + i] : (float)static_cast<const T*>(a.add)[from + i];
        const float* at = red + tok * PITCH + row;
        if (p.split == 1) {
            const float4 v = *reinterpret_cast<const float4*>(at);
            f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
        } else {
            float4 v[kInt4MaxSplit];
#pragma unroll
            for (int r = 0; r < kInt4MaxSplit; ++r)
                if (r < p.split) v[r] = remote_f32x4(smem_u32(at), r);
            f[0] = f[1] = f[2] = f[3] = 0.f;
#pragma unroll
            for (int r = 0; r < kInt4MaxSplit; ++r)
                if (r < p.split) { f[0] += v[r].x; f[1] += v[r].y; f[2] += v[r].z; f[3] += v[r].w; }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (col + i >= a.n_out) break;
            if (p.y_f32) static_cast<float*>(a.y)[to + i] = fmaf(f[i], Codes<T>::kInverse, g[i]);
            else static_cast<T*>(a.y)[to + i] = (T)fmaf(f[i], Codes<T>::kInverse, g[i]);
        }
    }
    if (p.split > 1) cluster_sync();                          // nobody leaves while its sums are read
}

}  // namespace

// Into how many parts the columns of a tile are cut: rounds of blocks over the GPU times the stages of a block, to which its start
// and end add about three more.
constexpr int kInt4Fixed = 3;
inline int int4_split(long long tiles, int stages, int at_once) {
    int best = 1;
    long long least = 0;
    for (int split = 1; split <= kInt4MaxSplit && (split == 1 || stages >= 2 * split); split *= 2) {
        const long long cost = (tiles * split + at_once - 1) / at_once * ((stages + split - 1) / split + kInt4Fixed);
        if (split == 1 || cost < least) { best = split; least = cost; }
    }
    return best;
}

// launch of a cluster of p.split blocks along y
template <auto KERNEL>
inline cudaError_t launch_int4_kernel(const Int4Params& p, dim3 grid, int threads, size_t smem, cudaStream_t s) {
    const cudaError_t e = allow_smem<KERNEL>();
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1; attr[1].val.clusterDim.y = (unsigned)p.split; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.split > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, KERNEL, p);
}

// Codes as 16-bit numbers [n_out, n_in / 4], boxes of 128 bytes by 128 rows.  x as panels of 64 columns where they divide
// its rows, `panels` of them in one copy, else panel by panel.
inline bool encode_int4(Int4Params& p, uint32_t tokens, uint32_t panels) {
    const b200_int4& a = p.a;
    const uint64_t k = a.n_in, t = a.n_tokens;
    p.x_panels = a.n_in % 64 == 0;
    return encode_map(&p.codes, a.codes, {k / 4, (uint64_t)a.n_out}, {k / 4}, {64, kTcRows}) &&
           (p.x_panels ? encode_map(&p.x, a.x, {64, t, k / 64}, {(uint64_t)a.x_row, 64}, {64, tokens, panels})
                       : encode_map(&p.x, a.x, {k, t}, {(uint64_t)a.x_row}, {64, tokens}));
}

bool int4_rows_take(const b200_int4& a);      // one or two tokens, as long as x fits and the product is not too large
cudaError_t launch_int4_rows(const b200_int4& a, int dtype, int y_f32, int n_sm, cudaStream_t s);
cudaError_t launch_int4_few(const b200_int4& a, int dtype, int y_f32, int n_sm, cudaStream_t s);      // up to kInt4Few tokens
// Eight tokens there and nine on the tensor core's 128 rows by 16 tokens (int4_linear.cu): 4096 rows of 4096 columns, groups of 128, 8.8
// and 8.0 us, 8192 of 8192 17.5 and 17.1 us; 1024 of 8192, groups of 32, 7.7 and 9.3 us, 32000 of 8192, groups of 64, 42 and 49 us.
constexpr int kInt4Few = 8;

}  // namespace b200lora
