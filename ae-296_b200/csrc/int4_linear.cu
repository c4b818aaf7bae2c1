// Products of a few tokens with 4-bit weights: y[t, n] = sum_g s[n, g] sum_{k in g} (c[n, k] - z[n, g]) x[t, k].
//
// Every weight is used for a few tokens only, so reading the codes bounds the kernel; next come the instructions that turn
// codes into numbers.  c - z is a whole number of at most five bits, exact in either 16-bit type, so a group's sum is left to
// the tensor core (128 weight rows by up to 64 tokens, fp32) and the scale is applied to that sum in fp32: nothing is
// rounded before y.
//
// A code becomes a number without a magic constant: four bits zero-extended to 16 are a subnormal number, and one
// multiply-add brings it to size and takes the zero point away (value c - z times a power of two that is taken
// back from the whole sum, where it cannot make a large scale infinite).  A 32-bit word of eight codes costs two logic operations, four byte permutations and four multiply-adds.
//
// A block takes 128 rows and a part of the columns.  Two threads copy codes (128 rows by 256 columns a stage) and x (128
// columns a block) by tensor copies; eight warps turn codes into 16-bit numbers, a lane per row, and store them to TMEM
// (through shared memory they would be written and read once more, and its bandwidth would bound the kernel); some threads issue
// the multiplications of a block of 128 columns, each group into TMEM columns of its own; four warps read those, a
// thread per row, and add them up with their scales.  Where the 128-row tiles alone are fewer than the SMs, a cluster of up to eight
// blocks shares a tile's columns and its sums are added through distributed shared memory in a fixed order.
// 8192 rows of 8192 columns, groups of 128, 64 tokens, added to y, bf16: 21 us (1.8 TB/s, 0.41 PFLOP/s; a simple mma.sync kernel took
// 103 us): 128 blocks have 16 stages each of some 2000 cycles.  Of these, turning codes into numbers needs 350 to 400 and the products 720, so
// it is the roles' waiting for one another that bounds a stage; which hand-over, has not been measured.
// Every wait is bounded: on expiry the outputs become NaN and `status` says so (tc_common.cuh).
#include "int4_common.cuh"

namespace b200lora {

namespace {

constexpr int kRows = kTcRows;
constexpr int kSumWarps = 4, kCodeWarps = 8;
constexpr int kCopyWarp = kSumWarps + kCodeWarps;             // of codes, and the next of x
constexpr int kMmaWarp = kCopyWarp + 2;                       // the first of Shape::kMmaWarps, which take the blocks in turns
constexpr int kStageK = 256, kBlockK = 128;
constexpr int kCodeStage = kRows * kStageK / 2;               // 16 KB
constexpr int kACols = kBlockK / 2;                           // TMEM columns of a block of numbers
constexpr int kRedPitch = kRows + 4;                          // floats of a token's sums
constexpr int kRing = 4;                                      // blocks of x
// Barriers of finished blocks.  Half of the code warps may wait for block b - 3 while block b + 1, the other half's, ends: on the
// same barrier that would be one round too many.
constexpr int kDone = 8;

// N: tokens of a block, G: columns of a group.  Few tokens: two blocks an SM share its memories.
template <int G, int N> struct Shape {
    static constexpr int kStages = N == 16 ? 5 : 8;           // of codes
    static constexpr int kX = N * kBlockK * 2;
    static constexpr int kBytes = kStages * kCodeStage + kRing * kX;
    static constexpr int kPer = kBlockK / G;                  // groups of a block
    static constexpr int kSumCols = kPer * N;                 // TMEM columns of a block's sums
    // blocks of sums and of numbers: as many as fit TMEM, of which two blocks an SM have half each
    static constexpr int kSumRoom = N == 16 ? (G == 32 ? 128 : 64) : 256;
    static constexpr int kSums = kSumRoom / kSumCols < 4 ? kSumRoom / kSumCols : 4;
    static constexpr int kNumbers = N == 16 ? (G == 32 ? 2 : 3) : 4;
    // A thread that waits for a barrier has waited for its last round too, or it could take the one before that for this one: the
    // threads that issue divide the blocks of sums, of numbers (kReady barriers for those) and of x.
    static constexpr int kMmaWarps = N == 16 || kSums == 2 ? 2 : 4;
    static constexpr int kReady = kNumbers == 3 ? 6 : kNumbers;
    static_assert(kSums % kMmaWarps == 0 && kReady % kMmaWarps == 0 && kReady % kNumbers == 0 && kRing % kMmaWarps == 0, "rounds in order");
    static constexpr int kThreads = (kMmaWarp + kMmaWarps) * 32;
    static constexpr int kUsed = kSums * kSumCols + kNumbers * kACols;
    static constexpr int kAlloc = kUsed <= 256 ? 256 : 512;
    static_assert(kSums >= 2 && kUsed <= (N == 16 ? 256 : 512), "TMEM of an SM has 512 columns");
    static_assert(N * kRedPitch * 4 <= kRing * kX, "the sums take x's place");
};
struct Int4Shared {
    unsigned long long codes_full[8], codes_empty[8], x_full[kRing], done[kDone], a_full[6], d_empty[4], drained;
    unsigned tmem, err;
    int codes_asked, x_asked;                                 // stages of codes and blocks of x that were requested
};

template <typename T, int G, int N>
__global__ void __launch_bounds__(Shape<G, N>::kThreads, N == 16 ? 2 : 1) int4_kernel(const __grid_constant__ Int4Params p) {
    extern __shared__ unsigned char smem_raw[];
    using S = Shape<G, N>;
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Int4Shared& sh = *reinterpret_cast<Int4Shared*>(smem + S::kBytes);
    const b200_int4& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row0 = blockIdx.x * kRows, part = blockIdx.y, tok0 = blockIdx.z * N;
    const int all = (a.n_in + kStageK - 1) / kStageK;
    const int s0 = (int)((long long)all * part / p.split), n_stages = (int)((long long)all * (part + 1) / p.split) - s0;
    const int n_blocks = 2 * n_stages, n_groups = a.n_in / G;
    constexpr int kPer = S::kPer;
    auto bar = [](unsigned long long& b) { return smem_u32(&b); };
    unsigned* err = &sh.err;
    const unsigned codes_at = smem_u32(smem), x_at = codes_at + S::kStages * kCodeStage;
    auto done = [&](int b, unsigned code) { return b < 0 || mbar_reached(bar(sh.done[b % kDone]), (b / kDone) & 1, err, code); };

    if (warp == kCopyWarp && lane == 0) {
        // the codes are on their way to L2 while the predecessor ends (what it may still write, L2 sees too)
        for (int s = 0; s < S::kStages && s < n_stages; ++s) prefetch_tensor(&p.codes, (s0 + s) * (kStageK / 4), row0);
        for (int i = 0; i < S::kStages; ++i) { mbar_init(bar(sh.codes_full[i]), 1); mbar_init(bar(sh.codes_empty[i]), kCodeWarps); }
        for (int i = 0; i < kRing; ++i) mbar_init(bar(sh.x_full[i]), 1);
        for (int i = 0; i < kDone; ++i) mbar_init(bar(sh.done[i]), 1);
        for (int i = 0; i < S::kReady; ++i) mbar_init(bar(sh.a_full[i]), kCodeWarps / 2);
        for (int i = 0; i < S::kSums; ++i) mbar_init(bar(sh.d_empty[i]), kSumWarps);
        mbar_init(bar(sh.drained), S::kMmaWarps);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        sh.err = 0u;
    }
    // TMEM only after the wait: a predecessor may let this block come before it has its own, and would then wait for this one's
    pdl_wait_prior();
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "n"(S::kAlloc) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = *reinterpret_cast<volatile unsigned*>(&sh.tmem);
    if (p.early && tid == 0) pdl_launch_dependents();

    float acc[N];                                             // of the summing threads
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;

    if (warp == kCopyWarp) {
        // ================= copies of codes =================
        if (lane == 0) {
            int s = 0;
            for (; s < n_stages; ++s) {
                const int slot = s % S::kStages;
                if (!mbar_reached(bar(sh.codes_empty[slot]), ((s / S::kStages) & 1) ^ 1, err, 1)) break;
                mbar_arrive_expect_tx(bar(sh.codes_full[slot]), kCodeStage);
                tensor_g2s_2d(codes_at + slot * kCodeStage, &p.codes, (s0 + s) * (kStageK / 4), row0, bar(sh.codes_full[slot]));
            }
            sh.codes_asked = s;
        }
        __syncwarp();
    } else if (warp == kCopyWarp + 1) {
        // ================= copies of x =================
        if (lane == 0) {
            int b = 0;
            for (; b < n_blocks; ++b) {
                const int at = b % kRing, k = s0 * kStageK + b * kBlockK;
                const unsigned dst = x_at + at * S::kX;
                if (!done(b - kRing, 2)) break;
                mbar_arrive_expect_tx(bar(sh.x_full[at]), S::kX);
                if (p.x_panels) tensor_g2s_3d(dst, &p.x, 0, tok0, k / 64, bar(sh.x_full[at]));
                else {
                    tensor_g2s_2d(dst, &p.x, k, tok0, bar(sh.x_full[at]));
                    tensor_g2s_2d(dst + S::kX / 2, &p.x, k + 64, tok0, bar(sh.x_full[at]));
                }
            }
            sh.x_asked = b;
        }
        __syncwarp();
    } else if (warp >= kMmaWarp) {
        // ================= multiplications: several threads, since one cannot wait and issue as fast as the tensor core =================
        if (lane == 0) {
            const unsigned idesc = idesc_of(Cvt<T>::is_bf16, N, false);
            for (int b = warp - kMmaWarp; b < n_blocks; b += S::kMmaWarps) {
                const int at = b % kRing, from = b % S::kNumbers, to = b % S::kSums;
                if (!mbar_reached(bar(sh.d_empty[to]), ((b / S::kSums) & 1) ^ 1, err, 3) ||
                    !mbar_reached(bar(sh.x_full[at]), (b / kRing) & 1, err, 4) ||
                    !mbar_reached(bar(sh.a_full[b % S::kReady]), (b / S::kReady) & 1, err, 5))
                    break;
                tc_fence_after();
                const unsigned xa = desc_low(x_at + at * S::kX, kRowsAreRows);
                const unsigned w = tmem + S::kSums * S::kSumCols + from * kACols, d = tmem + to * S::kSumCols;
#pragma unroll
                for (int i = 0; i < kBlockK / 16; ++i)
                    mma_ts(d + (i * 16 / G) * N, w + i * 8, xa + (((i >> 2) * (S::kX / 2) + (i & 3) * 32) >> 4), idesc, i % (G / 16) != 0);
                tc_commit(bar(sh.done[b % kDone]));
            }
        }
        __syncwarp();
    } else if (warp >= kSumWarps) {
        // ================= codes to numbers: a lane per row, a half of each stage =================
        const int cw = warp - kSumWarps, half = cw >> 2, row = (cw & 3) * 32 + lane;
        const int n_row = min(row0 + row, a.n_out - 1);
        const unsigned char* zeros = static_cast<const unsigned char*>(a.zeros) + (long long)n_row * n_groups;
        const unsigned lanes = (unsigned)((cw & 3) * 32) << 16;
        // The zeros of a half stage as the bytes of a word, three stages ahead.  Where words are not aligned (a number of
        // columns that 128 does not divide) they are read byte by byte.
        const bool words = n_groups % kPer == 0 && (reinterpret_cast<uintptr_t>(a.zeros) & (kPer - 1)) == 0;
        auto load_zeros = [&](int s) {
            const int gi = (s0 + s) * (kStageK / G) + half * kPer;
            unsigned z = 0u;
            if (!a.zeros) return 0x08080808u;
            if (s >= n_stages) return z;
            if (words) {
                if (gi < n_groups)
                    z = kPer == 4 ? __ldg(reinterpret_cast<const unsigned*>(zeros + gi)) : kPer == 2 ? __ldg(reinterpret_cast<const unsigned short*>(zeros + gi)) : __ldg(zeros + gi);
            } else
#pragma unroll
                for (int g = 0; g < kPer; ++g)
                    if (gi + g < n_groups) z |= (unsigned)__ldg(zeros + gi + g) << (8 * g);
            return z;
        };
        if (a.zeros && half == 0)                             // a row's zeros of this part are read a few bytes a stage: into L2 at once
            for (int g = s0 * (kStageK / G); g < min((s0 + n_stages) * (kStageK / G), n_groups); g += 32) prefetch_l2(zeros + g);
        unsigned z[3] = {load_zeros(0), load_zeros(1), load_zeros(2)};
        for (int s = 0; s < n_stages; ++s) {
            const int slot = s % S::kStages, b = 2 * s + half, at = b % S::kNumbers;
            unsigned offset[kPer];
#pragma unroll
            for (int g = 0; g < kPer; ++g) offset[g] = zero_offset<T>(z[0] >> (8 * g) & 15u);
            z[0] = z[1]; z[1] = z[2];
            z[2] = load_zeros(s + 3);
            // (If one of these expires, or a sum's, the tensor core multiplies what is not there yet, and y is NaN anyway.  Only a copy
            // may not be asked for while the stage's last one is under way.)
            mbar_reached(bar(sh.codes_full[slot]), (s / S::kStages) & 1, err, 6);
            done(b - S::kNumbers, 7);
            __syncwarp();                                     // lanes may leave a wait one by one: what follows is for whole warps
            tc_fence_after();
            const unsigned from = codes_at + slot * kCodeStage + row * 128;
            const unsigned to = tmem + lanes + S::kSums * S::kSumCols + at * kACols;
#pragma unroll
            for (int q = 0; q < 4; ++q) {                     // 32 columns
                unsigned w[4], v[16];
                lds16(from + (((half * 4 + q) ^ (row & 7)) << 4), w);
                const unsigned o = offset[q * 32 / G];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    unsigned e[4];
                    eight_columns<T>(w[j], o, e);
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[4 * j + i] = e[i];
                }
                tc_st16(to + q * 16, v);
            }
            if (lane == 0 && *reinterpret_cast<volatile unsigned*>(err) == 0u) mbar_arrive(bar(sh.codes_empty[slot]));
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(sh.a_full[b % S::kReady]));
        }
    } else {
        // ================= sums: a thread per row =================
        const int row = tid, n_row = min(row0 + row, a.n_out - 1);
        const unsigned short* scales = static_cast<const unsigned short*>(a.scales) + (long long)n_row * n_groups;
        const unsigned lanes = (unsigned)(warp * 32) << 16;
        // a block's scales as halves of two words, four blocks ahead (as the zeros above)
        const bool words = n_groups % kPer == 0 && (reinterpret_cast<uintptr_t>(a.scales) & (2 * kPer - 1)) == 0;
        auto load_scales = [&](int b) {
            const int gi = s0 * (kStageK / G) + b * kPer;
            uint2 v = make_uint2(0u, 0u);
            if (b >= n_blocks) return v;
            if (words) {
                if (gi < n_groups) {
                    if (kPer == 4) v = __ldg(reinterpret_cast<const uint2*>(scales + gi));
                    else if (kPer == 2) v.x = __ldg(reinterpret_cast<const unsigned*>(scales + gi));
                    else v.x = __ldg(scales + gi);
                }
            } else {
#pragma unroll
                for (int g = 0; g < kPer; ++g)
                    if (gi + g < n_groups) (g < 2 ? v.x : v.y) |= (unsigned)__ldg(scales + gi + g) << (16 * (g & 1));
            }
            return v;
        };
        for (int g = s0 * (kStageK / G); g < min((s0 + n_stages) * (kStageK / G), n_groups); g += 16) prefetch_l2(scales + g);
        uint2 sc[4] = {load_scales(0), load_scales(1), load_scales(2), load_scales(3)};
        for (int b = 0; b < n_blocks; ++b) {
            float f[kPer];
#pragma unroll
            for (int g = 0; g < kPer; ++g) f[g] = from_bits<T>((unsigned short)((g < 2 ? sc[0].x : sc[0].y) >> (16 * (g & 1))));
            sc[0] = sc[1]; sc[1] = sc[2]; sc[2] = sc[3];
            sc[3] = load_scales(b + 4);
            done(b, 8);
            __syncwarp();
            tc_fence_after();
            const unsigned d = tmem + lanes + (b % S::kSums) * S::kSumCols;
#pragma unroll
            for (int g = 0; g < kPer; ++g)
#pragma unroll
                for (int c = 0; c < N; c += 16) {
                    unsigned v[16];
                    tc_ld16(d + g * N + c, v);
                    tc_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[c + i] = fmaf(f[g], __uint_as_float(v[i]), acc[c + i]);
                }
            tc_fence_before();
            if (lane == 0) mbar_arrive(bar(sh.d_empty[b % S::kSums]));
        }
    }
    if (!p.early && tid == 0) pdl_launch_dependents();                    // late, as in int4_few.cu
    // ---- sums to shared memory, where x was (all multiplications are complete: they were summed)
    __syncthreads();
    const bool lost = *reinterpret_cast<volatile unsigned*>(err) != 0u;
    if (lost) {
        if (lane == 0) {
            if (warp >= kMmaWarp) {
                tc_commit(bar(sh.drained));
                mbar_drain(bar(sh.drained), 0);
            } else if (warp == kCopyWarp)
                for (int s = max(sh.codes_asked - S::kStages, 0); s < sh.codes_asked; ++s) mbar_drain(bar(sh.codes_full[s % S::kStages]), (s / S::kStages) & 1);
            else if (warp == kCopyWarp + 1)
                for (int b = max(sh.x_asked - kRing, 0); b < sh.x_asked; ++b) mbar_drain(bar(sh.x_full[b % kRing]), (b / kRing) & 1);
        }
        if (tid == 0 && a.status) atomicOr(a.status, B200_DECODE_TIMEOUT);
        __syncthreads();
    }
    float* red = reinterpret_cast<float*>(smem + S::kStages * kCodeStage);
    if (warp < kSumWarps) {
#pragma unroll
        for (int i = 0; i < N; ++i) red[i * kRedPitch + tid] = lost ? __int_as_float(0x7fffffff) : acc[i];
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::kAlloc) : "memory");
    finish_sums<T, N, kRedPitch, S::kThreads>(p, red, row0, tok0, part);
}

template <typename T, int G, int N>
cudaError_t launch_tokens(const b200_int4& a, int y_f32, int n_sm, cudaStream_t s) {
    Int4Params p;
    p.a = a; p.y_f32 = y_f32;
    if (!encode_int4(p, N, 2)) return cudaErrorInvalidValue;
    const int tiles = (a.n_out + kRows - 1) / kRows, stages = (a.n_in + kStageK - 1) / kStageK, blocks = (a.n_tokens + N - 1) / N;
    p.split = int4_split((long long)tiles * blocks, stages, n_sm);
    p.early = (long long)tiles * blocks * p.split <= n_sm;
    return launch_int4_kernel<int4_kernel<T, G, N>>(p, dim3((unsigned)tiles, (unsigned)p.split, (unsigned)blocks), Shape<G, N>::kThreads,
                              Shape<G, N>::kBytes + sizeof(Int4Shared) + 1024, s);
}
template <typename T, int G>
cudaError_t launch_group(const b200_int4& a, int y_f32, int n_sm, cudaStream_t s) {
    if (a.n_tokens <= 16) return launch_tokens<T, G, 16>(a, y_f32, n_sm, s);
    // sums of 64 tokens of four groups would leave no TMEM for the numbers
    if constexpr (G > 32)
        if (a.n_tokens > 32) return launch_tokens<T, G, 64>(a, y_f32, n_sm, s);
    return launch_tokens<T, G, 32>(a, y_f32, n_sm, s);
}
template <typename T>
cudaError_t launch_typed(const b200_int4& a, int y_f32, int n_sm, cudaStream_t s) {
    return a.group == 128 ? launch_group<T, 128>(a, y_f32, n_sm, s) : a.group == 64 ? launch_group<T, 64>(a, y_f32, n_sm, s) : launch_group<T, 32>(a, y_f32, n_sm, s);
}

}  // namespace

cudaError_t launch_int4(const b200_int4& a, int dtype, int y_f32, int n_sm, cudaStream_t s) {
    if (int4_rows_take(a)) return launch_int4_rows(a, dtype, y_f32, n_sm, s);
    if (a.n_tokens <= kInt4Few) return launch_int4_few(a, dtype, y_f32, n_sm, s);
    return dtype == B200_LORA_F16 ? launch_typed<__half>(a, y_f32, n_sm, s) : launch_typed<__nv_bfloat16>(a, y_f32, n_sm, s);
}

}  // namespace b200lora
