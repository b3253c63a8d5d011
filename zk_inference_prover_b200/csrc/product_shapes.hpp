// Products of codes: the shapes of their tiles, and what their parts wait for. Without a GPU's types, so that they can be looked at on the host.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define ZK_ON_DEVICE __device__ __forceinline__
#else
#define ZK_ON_DEVICE inline
#endif

namespace zk {

// RAW: 4-bit weights come to shared memory by the tensor memory unit (their rows start on 16-byte boundaries, and x's); x then has a ring of its own, longer than the codes' one.
template <bool INT4, int N, bool TMA>
struct Tile {
    static constexpr bool FILLED = INT4 || !TMA, RAW = INT4 && TMA;     // the weights' part of a stage is written by warps; from shared memory
    static constexpr int EPI = N == 64 ? (INT4 ? 8 : 4) : N >= 128 ? 8 : 4, SETS = RAW ? (N == 128 ? 1 : 2) : INT4 ? 2 : 4;  // warps that read the sums; sets of four warps that write codes, in turn
    // (as many sets as leave the registers in place: 1193 rows of 6744 x 1342 8-bit codes on odd boundaries 122 us by 4 sets and 167 by 2; 2001 of 4097 x 6145 4-bit ones 527 by 2 and 1532 by 4)
    static constexpr int FIRST_FILLER = EPI + (INT4 ? 4 : 3), THREADS = 32 * (FILLED ? FIRST_FILLER + 4 * SETS : EPI + 2);
    // A step's codes, in halves of 128 that are a matrix each: what a step costs whatever its codes, waits above all, is some 600 cycles of each of the warps that it goes through.
    static constexpr int CODES = INT4 ? 256 : 128, HALVES = CODES / 128, A_HALF = 128 * 128, B_HALF = N * 128;
    static constexpr int A = HALVES * A_HALF, B = HALVES * B_HALF, STAGE = RAW ? A : A + B, RAW_BYTES = 128 * CODES / 2;
    // thread blocks an SM (one where codes are written by warps: two leave too few registers, sixteen rows of 4096 x 32000 4-bit codes 45 us and 29 by one)
    static constexpr int BLOCKS = N <= 64 && !FILLED ? 2 : 1;
    static constexpr int JOIN = N <= (INT4 ? 64 : 32) ? N * 512 : 0;                 // a cluster's sums
    static constexpr int RAWS = !RAW ? 0 : N == 32 ? 4 : 3, XS = !RAW ? 0 : N == 32 ? 3 : 2;
    static constexpr int SCALES = INT4 ? 4 : 0, SCALE_BYTES = 128 * 16; // eight groups' scales of a tile's outputs
    static constexpr int ROOM = (BLOCKS == 2 ? 112 * 1024 : 216 * 1024) - JOIN - RAWS * RAW_BYTES - XS * B - SCALES * SCALE_BYTES;
    static constexpr int STAGES = ROOM / STAGE < 6 ? ROOM / STAGE : 6;
    // The sums of a tile of 8-bit weights, or of 4-bit weights' groups: of a step's all at once where they have room twice.
    static constexpr bool BY_STEP = INT4 && N == 32;
    static constexpr int SUMS = !INT4 || BY_STEP ? 2 : 4, SUM = BY_STEP ? 8 * N : N, COLUMNS = SUMS * SUM < 32 ? 32 : SUMS * SUM;
    // A thread block never waits for tensor memory: those that fit an SM's shared memory together (this kernel's variants and attention's, which take all columns and 121 KB) fit its
    // 512 columns. Clusters that each hold what another waits for would wait forever.
    static constexpr int LEAST = BLOCKS == 2 ? 108 * 1024 : 121 * 1024;
    static constexpr int USED = STAGES * STAGE + RAWS * RAW_BYTES + XS * B + SCALES * SCALE_BYTES + JOIN, SMEM = 1024 + (USED > LEAST ? USED : LEAST);
    static_assert(COLUMNS * BLOCKS <= 512 && (COLUMNS & (COLUMNS - 1)) == 0 && STAGES >= 2 && SMEM <= 226 * 1024, "");
    // A wait names the parity of a phase, so it has to know that the phase two before has ended. Sets of warps that write codes skip each other's steps: that the stage's codes before have been multiplied
    // says it of the weights that they came from where the ring of those is no shorter (before_codes), a set's own last wait says it of a stage, and of the ends of reads, of which there are 32 barriers.
    static_assert(!RAW || STAGES <= RAWS, "");
    static_assert(!FILLED || SETS <= STAGES, "");
    static_assert(!INT4 || (STAGES * (BY_STEP ? 1 : 8) <= 32 && SETS * (BY_STEP ? 1 : 8) < 32), "");
};

// What a set of warps waits for before it writes a step's codes into a stage: that the products of the step that was there before have ended, and then that this step's weights are in shared memory.
// In this order: with several sets another one has read the weights' place last, and copies may end in any order, so only the end of those products says that the copy before this one is there. Until
// it is, the barrier's parity is that of an older phase, and a wait for this one would be over at once.
template <class StageFree, class WeightsThere>
ZK_ON_DEVICE void before_codes(StageFree stage_free, WeightsThere weights_there) {
    stage_free();
    weights_there();
}

// Whether the scales of groups from `first` on, at address `at`, come eight at a time by 16 bytes: on their boundaries for every output (`stride` scales apart), and with nothing behind a row's last
// group, which of an array's last row is behind the array.
ZK_ON_DEVICE bool scales_by_eights(uintptr_t at, uint32_t first, uint32_t groups, int64_t stride, uint32_t n_out) {
    return at % 16 == 0 && (n_out == 1 || stride % 8 == 0) && first % 8 == 0 && groups % 8 == 0;
}

// Whether the two whole 16-byte blocks of memory that 16 bytes from p on lie in (the second one is taken with p on a boundary, too) reach out of the array [lo, hi).
ZK_ON_DEVICE bool blocks_reach_out(uintptr_t p, uintptr_t lo, uintptr_t hi) {
    const uintptr_t first = p - (p & 15);
    return first < lo || first + 32 > hi;
}

}  // namespace zk
