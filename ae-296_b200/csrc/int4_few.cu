// Products of three to eight tokens with 4-bit weights (see int4_linear.cu for the mathematics): mma.sync, 16 weight rows by eight
// tokens.  For so few tokens the tensor core of tcgen05 takes longer over a tile (45 cycles for 2048 weights, whatever the
// tokens) than the codes take to arrive; a warp's own multiplication takes 256 weights every three cycles and has its numbers
// in registers.
//
// A block of eight warps takes 128 rows and a part of the columns.  Codes (128 rows by 256 columns a stage) and x come by tensor
// copies; a warp waits for a stage by itself.  What a group needs besides, its scale in fp32 and the offset that takes zero
// point and base away, is made ready in shared memory for eight groups at a time, the next eight while these are multiplied.
//
// Seven tokens, bf16: 1024 rows of 8192 columns 7.5 us (64 blocks of four stages; copies, waits and the cluster's sums one after the
// other), 8192 rows 17.2 us, 32000 rows 42 us (3.4 TB/s): there the shared memory's bandwidth is used for half of the time and
// instructions issue for most of it.
#include "int4_common.cuh"

namespace b200lora {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = kTcRows;
constexpr int kTokens = kInt4Few;
constexpr int kStageK = 256;
constexpr int kCodeStage = kRows * kStageK / 2;               // 16 KB
constexpr int kXStage = kTokens * kStageK * 2;                // 4 KB
constexpr int kStages = 2;                                    // three blocks an SM have 96 KB of codes on their way
constexpr int kRedPitch = kRows + 4;

template <int G> struct Few {
    static constexpr int kChunkStages = G / 32;               // stages of a chunk
    static constexpr int kGroups = 8;                         // groups of a chunk
    static constexpr int kPitch = kGroups + 1;                // of a row, in pairs of words: rows a word pair apart in the banks
    static constexpr int kFactors = kRows * kPitch * 8;
    static constexpr int kBytes = kStages * (kCodeStage + kXStage) + 2 * kFactors;
};
struct FewShared {
    unsigned long long full[kStages], empty[kStages];
    unsigned err, pad;
};

// Of 128 columns a lane holds four words of eight: word j of lane t4 are the columns from 8 * column8(t4, j) on, all of
// one group for the words of one G / 32.
template <int G> __device__ __forceinline__ int column8(int t4, int j) {
    return G == 128 ? t4 * 4 + j : G == 64 ? (j >> 1) * 8 + t4 * 2 + (j & 1) : j * 4 + t4;
}

template <typename T, int G>
__global__ void __launch_bounds__(kThreads, 3) int4_few_kernel(const __grid_constant__ Int4Params p) {
    extern __shared__ unsigned char smem_raw[];
    using F = Few<G>;
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    FewShared& sh = *reinterpret_cast<FewShared*>(smem + F::kBytes);
    const b200_int4& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g4 = lane >> 2, t4 = lane & 3;
    const int row0 = blockIdx.x * kRows, part = blockIdx.y;
    const int all = (a.n_in + kStageK - 1) / kStageK;
    const int s0 = (int)((long long)all * part / p.split), n = (int)((long long)all * (part + 1) / p.split) - s0;
    const int n_groups = a.n_in / G;
    auto bar = [](unsigned long long& b) { return smem_u32(&b); };
    unsigned* err = &sh.err;
    const unsigned codes_at = smem_u32(smem), x_at = codes_at + kStages * kCodeStage;
    uint2* factors = reinterpret_cast<uint2*>(smem + kStages * (kCodeStage + kXStage));       // [2][rows][kPitch]

    auto request = [&](int s) {
        const int slot = s % kStages;
        const unsigned full = bar(sh.full[slot]), x = x_at + slot * kXStage;
        mbar_arrive_expect_tx(full, kCodeStage + kXStage);
        tensor_g2s_2d(codes_at + slot * kCodeStage, &p.codes, (s0 + s) * (kStageK / 4), row0, full);
        if (p.x_panels) tensor_g2s_3d(x, &p.x, 0, 0, (s0 + s) * (kStageK / 64), full);
        else
#pragma unroll
            for (int i = 0; i < 4; ++i) tensor_g2s_2d(x + i * (kXStage / 4), &p.x, (s0 + s) * kStageK + i * 64, 0, full);
    };
    if (tid == 0) {
        // the codes are on their way to L2 while the predecessor ends (what it may still write, L2 sees too)
        for (int s = 0; s < kStages && s < n; ++s) prefetch_tensor(&p.codes, (s0 + s) * (kStageK / 4), row0);
        for (int i = 0; i < kStages; ++i) { mbar_init(bar(sh.full[i]), 1); mbar_init(bar(sh.empty[i]), kWarps); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        sh.err = 0u;
    }
    pdl_wait_prior();
    if (p.early && tid == 0) pdl_launch_dependents();
    __syncthreads();
    int asked = min(kStages, n);                               // stages requested so far (thread 0)
    if (tid == 0)
        for (int s = 0; s < asked; ++s) request(s);
    // ---- factors of a chunk: a thread makes half a row's
    constexpr int kHalf = F::kGroups / 2, kChunkStages = F::kChunkStages;
    const int f_row = tid >> 1, f_first = (tid & 1) * kHalf;
    const long long f_at = (long long)min(row0 + f_row, a.n_out - 1) * n_groups;
    static_assert(kHalf == 4, "two words of scales and one of zeros");
    // (a part may begin in the middle of four groups)
    const bool words = n_groups % 4 == 0 && s0 * (kStageK / G) % 4 == 0 && (reinterpret_cast<uintptr_t>(a.scales) & 7) == 0 && (reinterpret_cast<uintptr_t>(a.zeros) & 3) == 0;
    const unsigned short* scales = static_cast<const unsigned short*>(a.scales) + f_at;
    const unsigned char* zeros = static_cast<const unsigned char*>(a.zeros) + f_at;
    uint2 sc;
    unsigned ze;
    auto load_factors = [&](int chunk) {
        const int g = (s0 + chunk * kChunkStages) * (kStageK / G) + f_first;
        sc = make_uint2(0u, 0u);
        ze = a.zeros ? 0u : 0x08080808u;
        if (chunk * kChunkStages >= n || g >= n_groups) return;
        if (words) {
            sc = __ldg(reinterpret_cast<const uint2*>(scales + g));
            if (a.zeros) ze = __ldg(reinterpret_cast<const unsigned*>(zeros + g));
        } else
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (g + i < n_groups) {
                    (i < 2 ? sc.x : sc.y) |= (unsigned)__ldg(scales + g + i) << (16 * (i & 1));
                    if (a.zeros) ze |= (unsigned)__ldg(zeros + g + i) << (8 * i);
                }
    };
    auto store_factors = [&](int chunk) {
        uint2* to = factors + ((chunk & 1) * kRows + f_row) * F::kPitch + f_first;
#pragma unroll
        for (int i = 0; i < kHalf; ++i)
            to[i] = make_uint2(__float_as_uint(from_bits<T>((unsigned short)((i < 2 ? sc.x : sc.y) >> (16 * (i & 1))))),
                               zero_offset<T>(ze >> (8 * i) & 15u));
    };
    load_factors(0);
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    bool fine = true;                                          // no wait of this thread has expired
    for (int s = 0; s < n; ++s) {
        if (s % kChunkStages == 0) {
            const int chunk = s / kChunkStages;
            store_factors(chunk);
            __syncthreads();                                   // (the other half of the factors is done with since the last one)
            load_factors(chunk + 1);
        }
        if (tid == 0 && s > 0 && s - 1 + kStages < n) {        // the stage before this one is soon done with by all warps
            fine = fine && mbar_reached(bar(sh.empty[(s - 1) % kStages]), ((s - 1) / kStages) & 1, err, 2);
            if (fine) request(asked++);
        }
        const int slot = s % kStages;
        fine = fine && mbar_reached(bar(sh.full[slot]), (s / kStages) & 1, err, 1);
        __syncwarp();
        const uint2* fa = factors + ((s / kChunkStages & 1) * kRows + warp * 16 + g4) * F::kPitch + (s % kChunkStages) * (kStageK / G);
        const uint2* fb = fa + 8 * F::kPitch;
        const unsigned ca = codes_at + slot * kCodeStage + (warp * 16 + g4) * 128, cb = ca + 8 * 128;
        const unsigned xa = x_at + slot * kXStage + g4 * 128;
#pragma unroll
        for (int b = 0; b < 2; ++b) {                          // 128 columns: 64 bytes of a row
            unsigned w0[4], w1[4];
            if constexpr (G == 128) {
                lds16(ca + (((b * 4 + t4) ^ g4) << 4), w0);
                lds16(cb + (((b * 4 + t4) ^ g4) << 4), w1);
            } else if constexpr (G == 64) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int at = (((b * 4 + h * 2 + (t4 >> 1)) ^ g4) << 4) + (t4 & 1) * 8;
                    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w0[2 * h]), "=r"(w0[2 * h + 1]) : "r"(ca + at) : "memory");
                    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w1[2 * h]), "=r"(w1[2 * h + 1]) : "r"(cb + at) : "memory");
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int at = (((b * 4 + j) ^ g4) << 4) + t4 * 4;
                    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w0[j]) : "r"(ca + at) : "memory");
                    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w1[j]) : "r"(cb + at) : "memory");
                }
            }
#pragma unroll
            for (int g = 0; g < 128 / G; ++g) {
                const uint2 q0 = fa[b * (128 / G) + g], q1 = fb[b * (128 / G) + g];
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < G / 32; ++w) {
                    const int j = g * (G / 32) + w, c = b * 16 + column8<G>(t4, j);           // eight columns of 256
                    unsigned x[4], v0[4], v1[4];
                    lds16(xa + (c >> 3) * (kTokens * 128) + (((c & 7) ^ g4) << 4), x);
                    eight_columns<T>(w0[j], q0.y, v0);
                    eight_columns<T>(w1[j], q1.y, v1);
                    Mma<T>::run(sum, v0[0], v1[0], v0[1], v1[1], x[0], x[1]);
                    Mma<T>::run(sum, v0[2], v1[2], v0[3], v1[3], x[2], x[3]);
                }
                const float f0 = __uint_as_float(q0.x), f1 = __uint_as_float(q1.x);
                acc[0] = fmaf(f0, sum[0], acc[0]); acc[1] = fmaf(f0, sum[1], acc[1]);
                acc[2] = fmaf(f1, sum[2], acc[2]); acc[3] = fmaf(f1, sum[3], acc[3]);
            }
        }
        __syncwarp();
        if (lane == 0 && fine) mbar_arrive(bar(sh.empty[slot]));
    }
    // A grid of more blocks than SMs lets a successor's come only now: earlier they would take places on the SMs that have fewer
    // blocks of this grid, and all SMs would have to wait for those (8192 columns, 32000 rows: 61 us instead of 44 us, back to back).
    if (!p.early && tid == 0) pdl_launch_dependents();
    // ---- sums to shared memory, where the codes were
    __syncthreads();
    float* red = reinterpret_cast<float*>(smem);
    const bool lost = *reinterpret_cast<volatile unsigned*>(err) != 0u;
    if (lost) {
        if (tid == 0) {
            for (int s = max(asked - kStages, 0); s < asked; ++s) mbar_drain(bar(sh.full[s % kStages]), (s / kStages) & 1);
            if (a.status) atomicOr(a.status, B200_DECODE_TIMEOUT);
        }
        __syncthreads();
    }
    float* at = red + t4 * 2 * kRedPitch + warp * 16 + g4;
#pragma unroll
    for (int i = 0; i < 4; ++i) at[(i & 1) * kRedPitch + (i >> 1) * 8] = lost ? __int_as_float(0x7fffffff) : acc[i];
    finish_sums<T, kTokens, kRedPitch, kThreads>(p, red, row0, 0, part);
}

template <typename T, int G>
cudaError_t launch_group(const b200_int4& a, int y_f32, int n_sm, cudaStream_t s) {
    Int4Params p;
    p.a = a; p.y_f32 = y_f32;
    if (!encode_int4(p, kTokens, kStageK / 64)) return cudaErrorInvalidValue;
    const int tiles = (a.n_out + kRows - 1) / kRows, stages = (a.n_in + kStageK - 1) / kStageK;
    p.split = int4_split(tiles, stages, 2 * n_sm);
    p.early = p.split > 1;
    return launch_int4_kernel<int4_few_kernel<T, G>>(p, dim3((unsigned)tiles, (unsigned)p.split), kThreads, Few<G>::kBytes + sizeof(FewShared) + 1024, s);
}
template <typename T>
cudaError_t launch_typed(const b200_int4& a, int y_f32, int n_sm, cudaStream_t s) {
    return a.group == 128 ? launch_group<T, 128>(a, y_f32, n_sm, s) : a.group == 64 ? launch_group<T, 64>(a, y_f32, n_sm, s) : launch_group<T, 32>(a, y_f32, n_sm, s);
}

}  // namespace

cudaError_t launch_int4_few(const b200_int4& a, int dtype, int y_f32, int n_sm, cudaStream_t s) {
    return dtype == B200_LORA_F16 ? launch_typed<__half>(a, y_f32, n_sm, s) : launch_typed<__nv_bfloat16>(a, y_f32, n_sm, s);
}

}  // namespace b200lora
