// Products of one or two tokens with 4-bit weights (see int4_linear.cu for the mathematics) without the tensor core: its smallest
// tile has eight tokens, and for fewer it is the way there, through shared memory and its layouts, that takes the time.
//
// A lane takes 32 columns of a row with one load, which all lie in one group, and a warp 1024 columns of four rows; the codes of its
// next step are on their way while it multiplies.  Codes become exact 16-bit numbers c - z (int4_common.cuh) and are multiplied with x
// as it is by the multiply-add of 16-bit factors and an fp32 sum, so that x needs no conversion.  x lies in shared memory in the
// order in which lanes ask for it.  Where rows are few a block's warps share their columns.
//
// This way of doing it takes some 2.3 instructions a code, which bound it (for 32000 rows of 8192 columns the bytes would take 22 us);
// 0.75 of them go through the integer pipe (with fp32 numbers made by permutations 2.1 did: 45 us instead of 40 us for those rows).  One
// token, bf16, back to back: 4096 rows of 4096 columns 4.7 us, 1024 of 8192 3.7 us, 8192 of 8192 12.1 us (2.9 TB/s), 32000 of 8192 40.1 us
// (3.6 TB/s).  Rows shared out evenly among the warps instead of four at a time: 5.2, 3.9, 13.5, 42.7 us; three blocks an SM: 6.6, 4.8, 18.9,
// 46.1 us.
#include "int4_common.cuh"

namespace b200lora {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 4;                                      // of a warp
constexpr int kBlocks = 2;                                    // of an SM
constexpr int kStep = 1024;                                   // columns of a warp

// sum + a.lo * b.lo + a.hi * b.hi: 16-bit factors, exact products, fp32 sums
template <typename T> __device__ __forceinline__ float dot2(unsigned a, unsigned b, float sum);
template <> __device__ __forceinline__ float dot2<__half>(unsigned a, unsigned b, float sum) {
    asm("{ .reg .b16 al, ah, bl, bh; mov.b32 {al, ah}, %1; mov.b32 {bl, bh}, %2; fma.rn.f32.f16 %0, al, bl, %0; fma.rn.f32.f16 %0, ah, bh, %0; }"
        : "+f"(sum) : "r"(a), "r"(b));
    return sum;
}
template <> __device__ __forceinline__ float dot2<__nv_bfloat16>(unsigned a, unsigned b, float sum) {
    asm("{ .reg .b16 al, ah, bl, bh; mov.b32 {al, ah}, %1; mov.b32 {bl, bh}, %2; fma.rn.f32.bf16 %0, al, bl, %0; fma.rn.f32.bf16 %0, ah, bh, %0; }"
        : "+f"(sum) : "r"(a), "r"(b));
    return sum;
}

// What a lane needs of a step: 32 columns of each row, their scales and zero points.
struct Step {
    uint4 codes[kRows];
    unsigned short scale[kRows];
    unsigned char zero[kRows];
};

struct RowParams {
    b200_int4 a;
    int y_f32, parts, steps;                                  // warps of a block that share a group of rows; steps of a row
};

template <typename T, int TOKENS>
__global__ void __launch_bounds__(kThreads, kBlocks) int4_rows_kernel(const __grid_constant__ RowParams p) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float sums[kWarps][kRows * TOKENS];
    const b200_int4& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int parts = p.parts, part = warp % parts, per_block = kWarps / parts;
    const int row_groups = (a.n_out - 1) / kRows + 1, n_groups = a.n_in / a.group, workers = gridDim.x * per_block;
    int rg = blockIdx.x * per_block + warp / parts;           // group of kRows rows
    const int s0 = p.steps * part / parts, n_steps = p.steps * (part + 1) / parts - s0;
    auto row_of = [&](int rg, int r) { return (long long)(rg * kRows + min(r, a.n_out - 1 - rg * kRows)); };
    auto codes_of = [&](int rg, int r, int col) { return static_cast<const unsigned char*>(a.codes) + row_of(rg, r) * (a.n_in / 2) + col / 2; };
    {
        // the first codes are on their way to L2 while the predecessor ends (what it may still write, L2 sees too)
        const int col = s0 * kStep + lane * 32;
        if (rg < row_groups && col < a.n_in)
#pragma unroll
            for (int r = 0; r < kRows; ++r) prefetch_l2(codes_of(rg, r, col));
    }
    pdl_wait_prior();
    if (tid == 0) pdl_launch_dependents();

    auto load = [&](Step& s, int rg, int step) {
        const int col = step * kStep + lane * 32;
        if (rg >= row_groups || col >= a.n_in) return;
        const int g = col / a.group;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            s.codes[r] = __ldcs(reinterpret_cast<const uint4*>(codes_of(rg, r, col)));
            const long long at = row_of(rg, r) * n_groups + g;
            s.scale[r] = __ldg(static_cast<const unsigned short*>(a.scales) + at);
            s.zero[r] = a.zeros ? __ldg(static_cast<const unsigned char*>(a.zeros) + at) : 8;
        }
    };
    Step next = {};
    load(next, rg, s0);
    // ---- x: 8 columns of lane l's 32 in step s at (s * 4 + those) * 32 + l
    {
        const int pieces = a.n_in / 8, room = p.steps * (kStep / 8);
        uint4* xs = reinterpret_cast<uint4*>(smem);
        for (int i = tid; i < pieces; i += kThreads) {
            const int to = (i & ~127) + (i & 3) * 32 + (i >> 2 & 31);
#pragma unroll
            for (int t = 0; t < TOKENS; ++t)
                xs[t * room + to] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + (long long)t * a.x_row + i * 8);
        }
    }
    __syncthreads();

    const unsigned x_at = smem_u32(smem) + lane * 16, x_token = p.steps * (kStep * 2);
    const int turns = (row_groups - 1) / workers + 1;         // the same for all warps: they may meet in each
    for (int turn = 0; turn < turns; ++turn, rg += workers) {
        float acc[kRows][TOKENS];
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
            for (int t = 0; t < TOKENS; ++t) acc[r][t] = 0.f;
        for (int i = 0; i < n_steps; ++i) {
            const Step now = next;
            const int step = s0 + i;
            if (i + 1 < n_steps) load(next, rg, step + 1);
            else load(next, rg + workers, s0);
            if (rg >= row_groups || step * kStep + lane * 32 >= a.n_in) continue;
            float sum[kRows][TOKENS];
            unsigned less[kRows];
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                less[r] = zero_offset<T>(now.zero[r] & 15u);
#pragma unroll
                for (int t = 0; t < TOKENS; ++t) sum[r][t] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {                     // eight columns
                unsigned v[kRows][4];
#pragma unroll
                for (int r = 0; r < kRows; ++r)
                    eight_columns<T>(j == 0 ? now.codes[r].x : j == 1 ? now.codes[r].y : j == 2 ? now.codes[r].z : now.codes[r].w, less[r], v[r]);
#pragma unroll
                for (int t = 0; t < TOKENS; ++t) {
                    unsigned x[4];
                    lds16(x_at + t * x_token + (step * 4 + j) * 512, x);
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int r = 0; r < kRows; ++r) sum[r][t] = dot2<T>(v[r][c], x[c], sum[r][t]);
                }
            }
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const float f = from_bits<T>(now.scale[r]);
#pragma unroll
                for (int t = 0; t < TOKENS; ++t) acc[r][t] = fmaf(f, sum[r][t], acc[r][t]);
            }
        }
        // ---- the lanes' sums, then those of the warps that share the rows
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
            for (int t = 0; t < TOKENS; ++t) {
#pragma unroll
                for (int o = 16; o; o >>= 1) acc[r][t] += __shfl_xor_sync(0xffffffffu, acc[r][t], o);
                if (lane == r * TOKENS + t) sums[warp][lane] = acc[r][t];
            }
        if (parts > 1) __syncthreads(); else __syncwarp();
        const int r = lane / TOKENS, t = lane % TOKENS, row0 = rg < row_groups ? rg * kRows : 0, row = row0 + r;
        if (part == 0 && r < kRows && rg < row_groups && r < a.n_out - row0) {
            float f = 0.f;
            for (int w = 0; w < parts; ++w) f += sums[warp + w][lane];
            const long long to = (long long)t * a.y_row + row, from = (long long)t * a.add_row + row;
            const float g = !a.add ? 0.f : p.y_f32 ? static_cast<const float*>(a.add)[from] : (float)static_cast<const T*>(a.add)[from];
            f = fmaf(f, Codes<T>::kInverse, g);
            if (p.y_f32) static_cast<float*>(a.y)[to] = f;
            else static_cast<T*>(a.y)[to] = (T)f;
        }
        if (parts > 1) __syncthreads(); else __syncwarp();    // the sums' places are free
    }
}

template <typename T, int TOKENS>
cudaError_t launch_tokens(const b200_int4& a, int y_f32, int n_sm, cudaStream_t s) {
    RowParams p;
    p.a = a; p.y_f32 = y_f32;
    p.steps = (a.n_in + kStep - 1) / kStep;
    const long long row_groups = (a.n_out + kRows - 1) / kRows, slots = kBlocks * n_sm;
    p.parts = 1;
    while (p.parts < kWarps && 2 * p.parts <= p.steps && (row_groups * 2 * p.parts + kWarps - 1) / kWarps <= slots) p.parts *= 2;
    const long long blocks = (row_groups * p.parts + kWarps - 1) / kWarps;
    const size_t smem = (size_t)TOKENS * p.steps * kStep * 2;
    const cudaError_t e = allow_smem<int4_rows_kernel<T, TOKENS>>();
    if (e != cudaSuccess) return e;
    return launch_pdl(int4_rows_kernel<T, TOKENS>, dim3((unsigned)(blocks < slots ? blocks : slots)), dim3(kThreads), smem, s, p);
}
template <typename T>
cudaError_t launch_typed(const b200_int4& a, int y_f32, int n_sm, cudaStream_t s) {
    return a.n_tokens == 1 ? launch_tokens<T, 1>(a, y_f32, n_sm, s) : launch_tokens<T, 2>(a, y_f32, n_sm, s);
}

}  // namespace

bool int4_rows_take(const b200_int4& a) {
    // Two blocks an SM each have x in shared memory.  Two tokens of 8192 columns: 1024 rows 4.7 us (int4_few.cu: 7.4 us), 8192 rows
    // 16.0 us (17.1), 32000 rows 48.5 us (42.0): there the start no longer counts.
    const long long steps = (a.n_in + kStep - 1) / kStep;
    return a.n_tokens <= 2 && a.n_tokens * steps * kStep * 2 <= 96 * 1024 && (a.n_tokens == 1 || (long long)a.n_in * a.n_out <= 1 << 27);
}
cudaError_t launch_int4_rows(const b200_int4& a, int dtype, int y_f32, int n_sm, cudaStream_t s) {
    return dtype == B200_LORA_F16 ? launch_typed<__half>(a, y_f32, n_sm, s) : launch_typed<__nv_bfloat16>(a, y_f32, n_sm, s);
}

}  // namespace b200lora
