// Products of a few tokens with 4-bit weights: y[t, n] = sum_g s[n, g] sum_{k in g} (c[n, k] - z[n, g]) x[t, k].
//
// Every weight is used for a few tokens only, so reading the codes bounds the kernel.  A warp multiplies 16 weight rows
// (the rows of the matrix instruction) by up to 8 NT tokens (its columns).  c - z is a whole number of at most five
// bits and exact in either 16-bit type, so the products are exact, a group's sum is kept in the instruction's
// fp32 accumulator and the scale is applied to it in fp32: nothing is rounded before y.
// The codes need no rearranging: four bits at distance 16 make a pair of 16-bit numbers with one logic operation
// (1024 + c, or 128 + c in bf16: the code becomes the low bits of a number whose exponent is fixed), pairs (k, k + 4) of
// eight neighbouring columns; x is brought into the same order by byte permutations.
#include "decode_common.cuh"
#include "lora_pipe.cuh"

namespace b200lora {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kBlockK = 128;           // columns of a warp's step

template <typename T> struct Magic;
template <> struct Magic<__half> {
    static constexpr unsigned kBase = 0x64006400u;             // 1024
    static __device__ __forceinline__ unsigned sub(unsigned a, unsigned b) {
        __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
        return *reinterpret_cast<unsigned*>(&r);
    }
};
template <> struct Magic<__nv_bfloat16> {
    static constexpr unsigned kBase = 0x43004300u;             // 128
    static __device__ __forceinline__ unsigned sub(unsigned a, unsigned b) {
        __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
        return *reinterpret_cast<unsigned*>(&r);
    }
};
// (w & 0x000f000f) | base
__device__ __forceinline__ unsigned and_or(unsigned w, unsigned base) {
    unsigned r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "r"(0x000f000fu), "r"(base));
    return r;
}

// Words of codes of one row that a lane holds of a step: 32 columns in runs of G / 4, run i of group i of the step
template <int G> struct Codes { unsigned w[4]; };
template <int G>
__device__ __forceinline__ void load_codes(const unsigned char* row, int k0, int n_in, int t4, Codes<G>& c) {
    constexpr int kWords = G / 32;             // a lane's words of a group
#pragma unroll
    for (int s = 0; s < kBlockK / G; ++s) {
        const int k = k0 + s * G + t4 * (G / 4);
        if (k0 + s * G < n_in) {
            const unsigned char* p = row + (k >> 1);
            if constexpr (kWords == 4) {
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
                c.w[0] = v.x; c.w[1] = v.y; c.w[2] = v.z; c.w[3] = v.w;
            } else if constexpr (kWords == 2) {
                const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
                c.w[2 * s] = v.x; c.w[2 * s + 1] = v.y;
            } else c.w[s] = __ldg(reinterpret_cast<const unsigned*>(p));
        } else {
#pragma unroll
            for (int i = 0; i < kWords; ++i) c.w[s * kWords + i] = 0u;
        }
    }
}

template <typename T, int G, int NT>
__global__ void __launch_bounds__(kThreads) int4_kernel(const __grid_constant__ b200_int4 a, int y_f32) {
    __shared__ float red[kWarps][NT * 8][17];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g4 = lane >> 2, t4 = lane & 3;
    pdl_wait_prior();
    if (tid == 0) pdl_launch_dependents();
    const int row0 = blockIdx.x * 16, tok0 = blockIdx.y * NT * 8;
    const int ra = min(row0 + g4, a.n_out - 1), rb = min(row0 + g4 + 8, a.n_out - 1);      // rows behind the last repeat it
    const unsigned char* codes = static_cast<const unsigned char*>(a.codes);
    const unsigned char *ca = codes + (long long)ra * (a.n_in / 2), *cb = codes + (long long)rb * (a.n_in / 2);
    const int n_groups = a.n_in / G;
    const T *sa = static_cast<const T*>(a.scales) + (long long)ra * n_groups, *sb = static_cast<const T*>(a.scales) + (long long)rb * n_groups;
    const unsigned char* zeros = static_cast<const unsigned char*>(a.zeros);
    const unsigned char *za = zeros + (long long)ra * n_groups, *zb = zeros + (long long)rb * n_groups;
    const T* x[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int tok = tok0 + i * 8 + g4;
        x[i] = tok < a.n_tokens ? static_cast<const T*>(a.x) + (long long)tok * a.x_row : nullptr;
    }
    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;

    const int steps = (a.n_in + kBlockK - 1) / kBlockK;
    Codes<G> wa, wb;
    if (warp < steps) {
        load_codes<G>(ca, warp * kBlockK, a.n_in, t4, wa);
        load_codes<G>(cb, warp * kBlockK, a.n_in, t4, wb);
    }
    for (int step = warp; step < steps; step += kWarps) {
        Codes<G> na, nb;
        if (step + kWarps < steps) {
            load_codes<G>(ca, (step + kWarps) * kBlockK, a.n_in, t4, na);
            load_codes<G>(cb, (step + kWarps) * kBlockK, a.n_in, t4, nb);
        }
#pragma unroll
        for (int s = 0; s < kBlockK / G; ++s) {
            const int k0 = step * kBlockK + s * G;
            if (k0 >= a.n_in) break;
            const int gi = k0 / G;
            const float fa = (float)sa[gi], fb = (float)sb[gi];
            const unsigned ma = Magic<T>::kBase + (zeros ? (za[gi] & 15u) * 0x00010001u : 0x00080008u);
            const unsigned mb = Magic<T>::kBase + (zeros ? (zb[gi] & 15u) * 0x00010001u : 0x00080008u);
            float part[NT][4];
#pragma unroll
            for (int i = 0; i < NT; ++i) part[i][0] = part[i][1] = part[i][2] = part[i][3] = 0.f;
#pragma unroll
            for (int w = 0; w < G / 32; ++w) {
                const int k = k0 + t4 * (G / 4) + w * 8;
                const unsigned ua = wa.w[s * (G / 32) + w], ub = wb.w[s * (G / 32) + w];
                unsigned pa[4], pb[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    pa[j] = Magic<T>::sub(and_or(ua >> (4 * j), Magic<T>::kBase), ma);
                    pb[j] = Magic<T>::sub(and_or(ub >> (4 * j), Magic<T>::kBase), mb);
                }
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const uint4 v = x[i] ? __ldg(reinterpret_cast<const uint4*>(x[i] + k)) : make_uint4(0u, 0u, 0u, 0u);
                    const unsigned x04 = __byte_perm(v.x, v.z, 0x5410), x15 = __byte_perm(v.x, v.z, 0x7632);
                    const unsigned x26 = __byte_perm(v.y, v.w, 0x5410), x37 = __byte_perm(v.y, v.w, 0x7632);
                    Mma<T>::run(part[i], pa[0], pb[0], pa[1], pb[1], x04, x15);
                    Mma<T>::run(part[i], pa[2], pb[2], pa[3], pb[3], x26, x37);
                }
            }
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                acc[i][0] += fa * part[i][0]; acc[i][1] += fa * part[i][1];
                acc[i][2] += fb * part[i][2]; acc[i][3] += fb * part[i][3];
            }
        }
        wa = na; wb = nb;
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        red[warp][i * 8 + t4 * 2][g4] = acc[i][0]; red[warp][i * 8 + t4 * 2 + 1][g4] = acc[i][1];
        red[warp][i * 8 + t4 * 2][g4 + 8] = acc[i][2]; red[warp][i * 8 + t4 * 2 + 1][g4 + 8] = acc[i][3];
    }
    __syncthreads();
    for (int i = tid; i < NT * 8 * 16; i += kThreads) {
        const int tok = tok0 + (i >> 4), n = row0 + (i & 15);
        if (tok >= a.n_tokens || n >= a.n_out) continue;
        float f = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) f += red[w][i >> 4][i & 15];
        const long long at = (long long)tok * a.y_row + n, add_at = (long long)tok * a.add_row + n;
        if (y_f32) {
            if (a.add) f += static_cast<const float*>(a.add)[add_at];
            static_cast<float*>(a.y)[at] = f;
        } else {
            if (a.add) f += (float)static_cast<const T*>(a.add)[add_at];
            static_cast<T*>(a.y)[at] = (T)f;
        }
    }
}

template <typename T, int G>
cudaError_t launch_group(const b200_int4& a, int y_f32, cudaStream_t s) {
    const unsigned rows = (unsigned)((a.n_out + 15) / 16);
    if (a.n_tokens <= 8) return launch_pdl(int4_kernel<T, G, 1>, dim3(rows, 1), kThreads, 0, s, a, y_f32);
    if (a.n_tokens <= 16) return launch_pdl(int4_kernel<T, G, 2>, dim3(rows, 1), kThreads, 0, s, a, y_f32);
    return launch_pdl(int4_kernel<T, G, 4>, dim3(rows, (unsigned)((a.n_tokens + 31) / 32)), kThreads, 0, s, a, y_f32);
}
template <typename T>
cudaError_t launch_typed(const b200_int4& a, int y_f32, cudaStream_t s) {
    return a.group == 128 ? launch_group<T, 128>(a, y_f32, s) : a.group == 64 ? launch_group<T, 64>(a, y_f32, s) : launch_group<T, 32>(a, y_f32, s);
}

}  // namespace

cudaError_t launch_int4(const b200_int4& a, int dtype, int y_f32, int n_sm, cudaStream_t s) {
    (void)n_sm;
    return dtype == B200_LORA_F16 ? launch_typed<__half>(a, y_f32, s) : launch_typed<__nv_bfloat16>(a, y_f32, s);
}

}  // namespace b200lora
