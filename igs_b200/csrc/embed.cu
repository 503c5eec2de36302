// igs_embed: rows of a table by token, times a scale.  igs_embed_grad: the table's gradient,
//   d_table[v] = scale * sum of dy[i] over the places i with tokens[i] == v,
// dense, zeros for rows without a token.
//
// The gradient goes by sorted tokens instead of atomics: a stable sort of (token, place) puts the
// places of one token next to each other in their own order, so every row is one sum in 32 bits
// with a fixed sequence and one rounding, the same bits on every run.
//   1. sort.  Up to RANK_MAX places: one kernel ranks every place against all keys.  More: least
//      significant digits first, up to 10 bits a pass (a codebook of a million rows needs two), or
//      the whole row as one digit where its counts fit shared memory.
//      Places without a token in the table drop out.
//   2. segments: the sorted places are cut into chunks of equal length whatever the tokens are
//      (one common token may own most of them).  A run of one token inside a chunk is finished
//      there; the sums of runs that cross a border go to the chunk's two partial rows ("head":
//      it came from the chunk before, "tail": it started here and goes on).  The same launch
//      writes the zero rows.
//   3. join: the partial rows of a crossing run are added in order.
#include <cooperative_groups.h>

#include "feature.cuh"

namespace igs {

constexpr int EMBED_THREADS = 128;
constexpr int SORT_THREADS = 256;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int SORT_PER_WARP = 128;                       // places a warp ranks, 32 at a time
constexpr int SORT_BLOCK = SORT_WARPS * SORT_PER_WARP;   // places a block ranks
constexpr int SORT_MAX_BITS = 10;
constexpr int SORT_MAX_DIGITS = 1 << SORT_MAX_BITS;
constexpr long long EMBED_MAX_PLACES = (1ll << 31) - (1ll << 20);  // places are 32-bit numbers in the sort
constexpr long long EMBED_MAX_ROWS = (1ll << 31) - 2;
constexpr long long EMBED_MAX_WIDTH = 1ll << 22;

struct Tokens {
    const void* ptr;
    int wide;          // 64-bit tokens
    int has_empty;
    long long empty;   // the token of a place that holds none
    long long rows;    // tokens are 0 .. rows - 1
};

constexpr uint32_t NO_ROW = 0xffffffffu;

__device__ __forceinline__ long long token_at(const Tokens& t, long long i) {
    return t.wide ? static_cast<const long long*>(t.ptr)[i] : (long long)static_cast<const int*>(t.ptr)[i];
}
// the table's row for a place, or NO_ROW
__device__ __forceinline__ uint32_t row_of(const Tokens& t, long long tok) {
    if (t.has_empty && tok == t.empty) return NO_ROW;
    return tok >= 0 && tok < t.rows ? (uint32_t)tok : NO_ROW;
}

// The pack sizes in bytes that the kernels move, the widest on whose boundary all rows start.
static int embed_pack_bytes(const void* a, const void* b, long long D, long long row_stride, size_t size) {
    for (size_t bytes : {size_t(16), size_t(4)})
        if (bytes > size && aligned_to(a, bytes) && aligned_to(b, bytes) && (size_t)D * size % bytes == 0 &&
            (size_t)row_stride * size % bytes == 0)
            return (int)bytes;
    return (int)size;
}

// log2 of the threads that share a row of `packs` packs: the narrowest power of two that covers
// it, a whole block at most
static int group_log(long long packs) {
    int g = 0;
    while (g < 7 && (1 << g) < packs) ++g;
    static_assert(EMBED_THREADS == 1 << 7, "a block is the widest group");
    return g;
}

// ---------------------------------------------------------------------------
// lookup
// ---------------------------------------------------------------------------
struct EmbedArgs {
    Tokens tokens;
    const void* table;
    void* out;
    long long n, D, row_stride;
    float scale;
};

// A group of 2^log_g threads copies R rows, U packs of V values a thread at a time: the R tokens, then
// R U independent loads in flight.  Bound by memory and by how many rows are on their way: 65536 rows
// of 1024 bf16 from a table of 16384 take 32 us, its bytes at a copy's rate 26.
template <typename T, int V, int R, int U>
__global__ void __launch_bounds__(EMBED_THREADS) embed_kernel(EmbedArgs a, int log_g) {
    const int g = 1 << log_g, lane = threadIdx.x & (g - 1);
    const long long i0 = ((long long)blockIdx.x * (EMBED_THREADS >> log_g) + (threadIdx.x >> log_g)) * R;
    uint32_t row[R];
    float none[R];  // what fills the row of a place without one
#pragma unroll
    for (int r = 0; r < R; ++r) {
        row[r] = NO_ROW;
        none[r] = 0.f;
        if (i0 + r < a.n) {
            const long long tok = token_at(a.tokens, i0 + r);
            row[r] = row_of(a.tokens, tok);
            // an empty place is zero; a token outside the table is an error that shows: NaN
            if (!(a.tokens.has_empty && tok == a.tokens.empty)) none[r] = __int_as_float(0x7fc00000);
        }
    }
    const int packs = (int)(a.D / V);
    for (int p0 = lane; p0 < packs; p0 += g * U) {
        Pack<T, V> v[R][U];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const Pack<T, V>* src = reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(a.table) + (long long)row[r] * a.row_stride);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (row[r] != NO_ROW && p0 + u * g < packs) v[r][u] = src[p0 + u * g];
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (i0 + r >= a.n) continue;
            Pack<T, V>* out = reinterpret_cast<Pack<T, V>*>(static_cast<T*>(a.out) + (i0 + r) * a.D);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (p0 + u * g >= packs) continue;
                const Vals<V> y = row[r] != NO_ROW ? mul(to_vals<T, V>(v[r][u]), splat<V>(a.scale)) : splat<V>(none[r]);
                out[p0 + u * g] = to_pack<T, V>(y);
            }
        }
    }
}

template <typename T, int V>
static void launch_embed(const EmbedArgs& a, int device, cudaStream_t s) {
    // Four loads in flight a thread (with two or eight 65536 rows of 1024 bf16 took 6 and 23 % longer): of
    // four rows where a row has one pack a thread, of two rows where it has more (four of one row: 60000
    // rows of 514 bf16 took a third longer).  Rows go several to a group once that still
    // leaves every SM sixteen blocks; below, latency counts.
    constexpr int MOST = 4;
    const int log_g = group_log(a.D / V);
    const long long groups = EMBED_THREADS >> log_g;
    const bool wide = a.D / V > EMBED_THREADS, many = a.n >= (long long)sm_count(device) * 16 * groups * MOST;
    const long long per = groups * (!many ? 1 : wide ? 2 : MOST);
    const unsigned grid = (unsigned)((a.n + per - 1) / per);
    if (wide && many) embed_kernel<T, V, 2, 2><<<grid, EMBED_THREADS, 0, s>>>(a, log_g);
    else if (wide) embed_kernel<T, V, 1, MOST><<<grid, EMBED_THREADS, 0, s>>>(a, log_g);
    else if (many) embed_kernel<T, V, MOST, 1><<<grid, EMBED_THREADS, 0, s>>>(a, log_g);
    else embed_kernel<T, V, 1, 1><<<grid, EMBED_THREADS, 0, s>>>(a, log_g);
}

// ---------------------------------------------------------------------------
// sort
// ---------------------------------------------------------------------------
struct SortArgs {
    Tokens tokens;
    uint32_t* keys[2];  // in and out of the passes in turn; the first pass reads the tokens
    int* places[2];
    int* hist;          // [digits][blocks]: how often each block meets a digit, then its first slot in the digit
    int* totals;        // [digits]
    int* count;         // how many places hold a token
    long long n;
    int passes, bits;   // digits of `bits` bits
};

// Few places: every place's slot is the number of keys below its own plus the number of equal ones
// before it, counted over all keys.  Block b ranks the places 32 b .. 32 b + 31, one a lane; each
// warp counts over a share of the keys.  n^2 comparisons, but one launch and no passes: the 67 million
// of 8192 places take about 12 us over the whole device, the passes below 20.
__device__ __forceinline__ void count_below(int& n, uint32_t key, uint32_t below) {
    // (a predicated add; from `n += key < below` the compiler made five instructions)
    asm("{\n\t.reg .pred p;\n\tsetp.lt.u32 p, %1, %2;\n\t@p add.s32 %0, %0, 1;\n\t}" : "+r"(n) : "r"(key), "r"(below));
}
constexpr int RANK_MAX = 8192;
constexpr int RANK_WARPS = 16;
__global__ void __launch_bounds__(RANK_WARPS * 32) sort_rank_kernel(SortArgs a) {
    __shared__ __align__(16) uint32_t s_key[RANK_MAX];
    __shared__ int s_rank[RANK_WARPS][32];
    __shared__ int s_held[RANK_WARPS];
    let_next_start();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n = (int)a.n, padded = (n + 31) / 32 * 32;
    int held = 0;
    for (int i0 = 0; i0 < padded; i0 += RANK_WARPS * 32 * 8) {  // (eight loads on their way together)
        long long tok[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = i0 + j * (RANK_WARPS * 32) + threadIdx.x;
            if (i < n) tok[j] = token_at(a.tokens, i);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = i0 + j * (RANK_WARPS * 32) + threadIdx.x;
            const uint32_t k = i < n ? row_of(a.tokens, tok[j]) : NO_ROW;
            if (i < padded) s_key[i] = k;
            held += k != NO_ROW;
        }
    }
    __syncthreads();
    const int mine = blockIdx.x * 32 + lane;
    const uint32_t key = s_key[mine < padded ? mine : 0];
    const int tiles = padded / 32, per = (tiles + RANK_WARPS - 1) / RANK_WARPS;
    const int t1 = (warp + 1) * per < tiles ? (warp + 1) * per : tiles;
    int rank = 0;
    for (int t = warp * per; t < t1; ++t) {
        const uint4* tile = reinterpret_cast<const uint4*>(s_key + t * 32);
        if (t == blockIdx.x) {  // the block's own places: equal keys count when they come before
            for (int j = 0; j < 32; ++j) rank += s_key[t * 32 + j] < key + (j < lane ? 1u : 0u);
        } else {
            const uint32_t below = key + (t < (int)blockIdx.x ? 1u : 0u);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint4 k = tile[j];
                count_below(rank, k.x, below);
                count_below(rank, k.y, below);
                count_below(rank, k.z, below);
                count_below(rank, k.w, below);
            }
        }
    }
    s_rank[warp][lane] = rank;
    if (blockIdx.x == 0) {
        held = __reduce_add_sync(0xffffffffu, held);
        if (lane == 0) s_held[warp] = held;
    }
    __syncthreads();
    if (warp) return;
    int slot = 0;
#pragma unroll
    for (int w = 0; w < RANK_WARPS; ++w) slot += s_rank[w][lane];
    if (mine < n && key != NO_ROW) {
        a.keys[0][slot] = key;
        a.places[0][slot] = mine;
    }
    if (blockIdx.x == 0 && lane == 0) {
        int sum = 0;
        for (int w = 0; w < RANK_WARPS; ++w) sum += s_held[w];
        *a.count = sum;
    }
}

// More places: all passes in one cooperative launch.  (Three chained launches a pass take 3 us less on
// the device, 18 instead of 21 for 65536 places and two passes, but every launch costs the host 4: forward
// and gradient of 9000 places of width 32 take 52 us this way and 71 that.)  Block b owns a range of
// neighbouring positions.  A pass: it counts the digits of its range; once all have, it finds from the
// counts where each digit of its range goes (behind all smaller digits, and behind the same digit of
// the blocks before); then it ranks its range in order, 32 positions a warp at a time, and writes the
// pairs.
__global__ void __launch_bounds__(SORT_THREADS) sort_kernel(SortArgs a) {
    __shared__ int s_first[SORT_MAX_DIGITS];             // counts, then the next slot per digit
    __shared__ int s_warp[SORT_WARPS][SORT_MAX_DIGITS];  // per warp: counts, then first slots
    __shared__ int s_sum[SORT_WARPS];
    constexpr int PER = SORT_PER_WARP / 32;
    const auto grid = cooperative_groups::this_grid();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, blocks = (int)gridDim.x;
    const int digits = 1 << a.bits;

    for (int pass = 0; pass < a.passes; ++pass) {
        const uint32_t* keys_in = a.keys[(pass & 1) ^ 1];
        const int* places_in = a.places[(pass & 1) ^ 1];
        uint32_t* keys_out = a.keys[pass & 1];
        int* places_out = a.places[pass & 1];
        const int shift = pass * a.bits;
        const long long count = pass ? *a.count : a.n;
        const long long tiles = (count + SORT_BLOCK - 1) / SORT_BLOCK, each = (tiles + blocks - 1) / blocks;
        const long long from = blockIdx.x * each * SORT_BLOCK;
        const long long to = from + each * SORT_BLOCK < count ? from + each * SORT_BLOCK : count;
        // position i of the pass's input; NO_ROW when there is none
        const auto key_at = [&](long long i) {
            if (i >= to) return NO_ROW;
            return pass ? keys_in[i] : row_of(a.tokens, token_at(a.tokens, i));
        };
        const auto digit = [&](uint32_t key) { return (int)(key >> shift) & (digits - 1); };

        for (int d = threadIdx.x; d < digits; d += SORT_THREADS) s_first[d] = 0;
        __syncthreads();
        for (long long t = from; t < to; t += SORT_BLOCK) {
            uint32_t key[SORT_BLOCK / SORT_THREADS];
#pragma unroll
            for (int j = 0; j < SORT_BLOCK / SORT_THREADS; ++j) key[j] = key_at(t + j * SORT_THREADS + threadIdx.x);
#pragma unroll
            for (int j = 0; j < SORT_BLOCK / SORT_THREADS; ++j)
                // (integer counts: the result does not depend on the order of the adds)
                if (key[j] != NO_ROW) atomicAdd(&s_first[digit(key[j])], 1);
        }
        __syncthreads();
        for (int d = threadIdx.x; d < digits; d += SORT_THREADS) a.hist[(long long)d * blocks + blockIdx.x] = s_first[d];
        grid.sync();

        // a warp per digit, dealt out over the blocks: exclusive sums over the blocks, and the total
        for (int d = blockIdx.x + warp * blocks; d < digits; d += SORT_WARPS * blocks) {
            int* h = a.hist + (long long)d * blocks;
            int run = 0;
            for (int b0 = 0; b0 < blocks; b0 += 32) {
                const int b = b0 + lane, v = b < blocks ? h[b] : 0;
                int incl = v;
#pragma unroll
                for (int s = 1; s < 32; s <<= 1) {
                    const int t = __shfl_up_sync(0xffffffffu, incl, s);
                    if (lane >= s) incl += t;
                }
                if (b < blocks) h[b] = run + incl - v;
                run += __shfl_sync(0xffffffffu, incl, 31);
            }
            if (lane == 0) a.totals[d] = run;
        }
        grid.sync();

        // first slots of this block's digits: exclusive sums of the totals, four neighbours a thread
        constexpr int DIGITS = SORT_MAX_DIGITS / SORT_THREADS;
        int c[DIGITS], h[DIGITS], sum = 0;
#pragma unroll
        for (int j = 0; j < DIGITS; ++j) {
            const int d = threadIdx.x * DIGITS + j;
            c[j] = d < digits ? a.totals[d] : 0;
            h[j] = d < digits ? a.hist[(long long)d * blocks + blockIdx.x] : 0;
            sum += c[j];
        }
        int incl = sum;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, s);
            if (lane >= s) incl += v;
        }
        if (lane == 31) s_sum[warp] = incl;
        __syncthreads();
        int run = incl - sum;
        for (int w = 0; w < warp; ++w) run += s_sum[w];
#pragma unroll
        for (int j = 0; j < DIGITS; ++j) {
            const int d = threadIdx.x * DIGITS + j;
            if (d < digits) s_first[d] = run + h[j];
            run += c[j];
        }
        if (pass == 0 && blockIdx.x == 0 && threadIdx.x == SORT_THREADS - 1) *a.count = run;
        __syncthreads();

        for (long long t = from; t < to; t += SORT_BLOCK) {  // (the same for the whole block)
            uint32_t key[PER];
            int place[PER], rank[PER];
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const long long i = t + warp * SORT_PER_WARP + j * 32 + lane;
                key[j] = key_at(i);
                place[j] = pass && i < to ? places_in[i] : (int)i;
            }
            for (int d = lane; d < digits; d += 32) s_warp[warp][d] = 0;
            __syncwarp();
            // rank within the warp, in order of position
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const bool ok = key[j] != NO_ROW;
                // what is not there shares a digit no pair has, and so matches only its like
                const int d = ok ? digit(key[j]) : SORT_MAX_DIGITS;
                const unsigned peers = __match_any_sync(0xffffffffu, d);
                const int before = __popc(peers & ((1u << lane) - 1u));
                rank[j] = ok ? s_warp[warp][d] + before : 0;
                __syncwarp();
                if (ok && before == 0) s_warp[warp][d] += __popc(peers);
                __syncwarp();
            }
            __syncthreads();
            for (int d = threadIdx.x; d < digits; d += SORT_THREADS) {
                int slot = s_first[d];
#pragma unroll
                for (int w = 0; w < SORT_WARPS; ++w) {
                    const int n = s_warp[w][d];
                    s_warp[w][d] = slot;
                    slot += n;
                }
                s_first[d] = slot;
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                if (key[j] == NO_ROW) continue;
                const long long slot = s_warp[warp][digit(key[j])] + rank[j];
                // slot < n by construction; the guard keeps a corrupted workspace from turning into a stray write
                if (slot >= 0 && slot < a.n) {
                    keys_out[slot] = key[j];
                    places_out[slot] = place[j];
                }
            }
            __syncthreads();
        }
        if (pass + 1 < a.passes) grid.sync();
    }
    let_next_start();
}

// Codebooks of 1025 to 16384 rows and one tile a block: one pass, a digit being the whole row.  The
// blocks' counts are [blocks][rows]; a thread per row sums its column over the blocks.  A block's 1024
// pairs are ranked without any order between warps: an entry of 32 bits per row holds the counts of four
// warps in a byte each (a warp has 128 pairs), first of warps 0 to 3, then of 4 to 7.  (64 bits would do it
// in one round, 1 us sooner, but with 64 KB a block two calls' blocks fit an SM together.)  Whole gradient
// issued eagerly, two passes as above against this: 27696 places of 5003 x 771 fp32 68 and 63 us, 65536 of 16384 x 1024 bf16
// 67 and 65, 131072 of 2000 x 64 57 and 51, 9000 of 16384 x 64 35 and 37.
constexpr int WIDE_MAX_BITS = 14;
__global__ void __launch_bounds__(SORT_THREADS) sort_wide_kernel(SortArgs a) {
    extern __shared__ __align__(16) unsigned char s_mem[];
    __shared__ int s_sum[SORT_WARPS], s_base[(1 << WIDE_MAX_BITS) / SORT_THREADS];
    constexpr int PER = SORT_PER_WARP / 32;
    static_assert(SORT_WARPS == 8 && SORT_PER_WARP < 256, "a byte a warp, two rounds");
    const auto grid = cooperative_groups::this_grid();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, blocks = (int)gridDim.x;
    const int digits = 1 << a.bits;
    int* s_count = reinterpret_cast<int*>(s_mem);            // [digits]
    unsigned* s_ranks = reinterpret_cast<unsigned*>(s_mem);  // [digits], later
    int* mine = a.hist + (long long)blockIdx.x * digits;     // this block's counts, then first slots

    const long long first = (long long)blockIdx.x * SORT_BLOCK + warp * SORT_PER_WARP + lane;
    uint32_t key[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) key[j] = first + j * 32 < a.n ? row_of(a.tokens, token_at(a.tokens, first + j * 32)) : NO_ROW;
    for (int d = threadIdx.x; d < digits / 4; d += SORT_THREADS) reinterpret_cast<int4*>(s_count)[d] = make_int4(0, 0, 0, 0);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j)
        if (key[j] != NO_ROW) atomicAdd(&s_count[key[j]], 1);  // (integer counts: no order changes the result)
    __syncthreads();
    for (int d = threadIdx.x; d < digits / 4; d += SORT_THREADS) reinterpret_cast<int4*>(mine)[d] = reinterpret_cast<int4*>(s_count)[d];
    grid.sync();

    // a thread per row: exclusive sums over the blocks; then over the rows of a group of SORT_THREADS
    int* group_sums = a.totals + digits;
    for (int d0 = blockIdx.x * SORT_THREADS; d0 < digits; d0 += blocks * SORT_THREADS) {
        int* column = a.hist + d0 + threadIdx.x;
        int run = 0;
        constexpr int U = 16;  // loads on their way together
        for (int b0 = 0; b0 < blocks; b0 += U) {
            int v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = b0 + u < blocks ? column[(long long)(b0 + u) * digits] : 0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (b0 + u < blocks) column[(long long)(b0 + u) * digits] = run;
                run += v[u];
            }
        }
        int incl = run;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, incl, s);
            if (lane >= s) incl += t;
        }
        if (lane == 31) s_sum[warp] = incl;
        __syncthreads();
        for (int w = 0; w < warp; ++w) incl += s_sum[w];
        a.totals[d0 + threadIdx.x] = incl - run;
        if (threadIdx.x == SORT_THREADS - 1) group_sums[d0 / SORT_THREADS] = incl;
        __syncthreads();
    }
    grid.sync();

    // where this block's pairs of a row go: behind the groups before, the rows before in the group, and
    // the same row in the blocks before
    int slot[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        slot[j] = key[j] != NO_ROW ? mine[key[j]] + a.totals[key[j]] : 0;
        if (key[j] != NO_ROW) s_ranks[key[j]] = 0;
    }
    const int groups = digits / SORT_THREADS;
    if (warp == 0) {
        int run = 0;
        for (int g0 = 0; g0 < groups; g0 += 32) {
            const int v = g0 + lane < groups ? group_sums[g0 + lane] : 0;
            int incl = v;
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const int t = __shfl_up_sync(0xffffffffu, incl, s);
                if (lane >= s) incl += t;
            }
            if (g0 + lane < groups) s_base[g0 + lane] = run + incl - v;
            run += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (blockIdx.x == 0 && lane == 0) *a.count = run;
    }
    const int half = warp / 4, shift = 8 * (warp % 4);
#pragma unroll
    for (int round = 0; round < 2; ++round) {
        __syncthreads();
        if (half == round) {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const unsigned peers = __match_any_sync(0xffffffffu, key[j]);
                const int before = __popc(peers & ((1u << lane) - 1u)), leader = __ffs(peers) - 1;
                unsigned old = 0;
                if (key[j] != NO_ROW && lane == leader) old = atomicAdd(&s_ranks[key[j]], (unsigned)__popc(peers) << shift);
                old = __shfl_sync(0xffffffffu, old, leader);
                slot[j] += (int)(old >> shift & 255u) + before;  // (only this warp adds to its byte)
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            if (key[j] == NO_ROW || half < round) continue;
            // the round's warps that come before this one
            const unsigned counts = s_ranks[key[j]] & (half == round ? (1u << shift) - 1u : 0xffffffffu);
            slot[j] += (int)__dp4a(counts, 0x01010101u, 0u);
        }
        if (round == 0) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (key[j] != NO_ROW) s_ranks[key[j]] = 0;
        }
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (key[j] == NO_ROW) continue;
        const long long at = (long long)s_base[key[j] / SORT_THREADS] + slot[j];
        // at < n by construction; the guard keeps a corrupted workspace from turning into a stray write
        if (at >= 0 && at < a.n) {
            a.keys[0][at] = key[j];
            a.places[0][at] = (int)(first + j * 32);
        }
    }
    let_next_start();
}

// ---------------------------------------------------------------------------
// sums over runs of one token
// ---------------------------------------------------------------------------
struct SegmentArgs {
    const uint32_t* keys;   // sorted
    const int* places;
    const int* count;       // how many
    const void* dy;
    void* d_table;
    float* part;            // [chunks][2][D]: head and tail sums
    long long rows, D;
    float scale;
    int chunks;
    int sum_blocks;         // blocks of the segment kernel that sum; the others write zero rows
    int log_g;              // a chunk is summed by 2^log_g threads a slab of columns
};

constexpr int CHUNK_STEP = 8;  // places whose rows are loaded together; chunks are multiples of it
// Steps of rows in a thread's ring, the one being added included.  16-bit values one by one cannot be
// copied asynchronously.
constexpr int SEGMENT_STAGES = 3;
template <typename T, int V>
constexpr bool segment_async = sizeof(Pack<T, V>) >= 4;
// Packs of columns a thread: one of 16 bytes, or four small ones (a group's width apart).
template <typename T, int V>
constexpr int segment_items = sizeof(Pack<T, V>) == 16 ? 1 : 4;
template <typename T, int V>
constexpr size_t segment_smem =
    segment_async<T, V> ? sizeof(Pack<T, V>) * segment_items<T, V> * CHUNK_STEP * SEGMENT_STAGES * EMBED_THREADS : 0;

// positions a chunk holds, the last one's less
__device__ __forceinline__ long long chunk_length(long long count, int chunks) {
    return ((count + chunks - 1) / chunks + CHUNK_STEP - 1) / CHUNK_STEP * CHUNK_STEP;
}

// whether a row has a token: binary search
__device__ __forceinline__ bool has_key(const uint32_t* keys, int count, uint32_t row) {
    int lo = 0, hi = count;
    while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        if (keys[mid] < row) lo = mid + 1; else hi = mid;
    }
    return lo < count && keys[lo] == row;
}

// sum * scale to a pack of a row of the table
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* row, long long pack, const Vals<V>& sum, float scale) {
    reinterpret_cast<Pack<T, V>*>(row)[pack] = to_pack<T, V>(mul(sum, splat<V>(scale)));
}

// grid (sum blocks + zero blocks, column slabs).  Every thread owns its packs of V columns and copies the
// rows of the next steps to shared memory of its own ahead of time: rows lie anywhere in dy, and what
// bounds the kernel is how many of them are on their way (plain loads, eight a thread between
// additions: 85 us for 65536 rows of 1024 bf16; the ring: 35).
template <typename T, int V>
__global__ void __launch_bounds__(EMBED_THREADS) segment_kernel(SegmentArgs a) {
    constexpr int ITEMS = segment_items<T, V>;
    let_next_start();
    wait_for_previous();
    const int count = *a.count, g = 1 << a.log_g;
    T* d_table = static_cast<T*>(a.d_table);
    const int packs = (int)(a.D / V), first_pack = (int)blockIdx.y * g * ITEMS;
    if ((int)blockIdx.x >= a.sum_blocks) {
        // rows without a token: a warp looks up 32 rows at a time, then writes those that have none
        const int lane = threadIdx.x & 31, last_pack = first_pack + g * ITEMS < packs ? first_pack + g * ITEMS : packs;
        const long long warps = (long long)(gridDim.x - a.sum_blocks) * (EMBED_THREADS / 32);
        const Pack<T, V> zero = to_pack<T, V>(splat<V>(0.f));
        for (long long r0 = ((long long)(blockIdx.x - a.sum_blocks) * (EMBED_THREADS / 32) + (threadIdx.x >> 5)) * 32;
             r0 < a.rows; r0 += warps * 32) {
            const long long r = r0 + lane;
            unsigned absent = __ballot_sync(0xffffffffu, r < a.rows && !has_key(a.keys, count, (uint32_t)r));
            while (absent) {
                const int k = __ffs(absent) - 1;
                absent &= absent - 1;
                Pack<T, V>* row = reinterpret_cast<Pack<T, V>*>(d_table + (r0 + k) * a.D);
                for (int p = first_pack + lane; p < last_pack; p += 32) row[p] = zero;
            }
        }
        return;
    }
    const long long chunk = (long long)blockIdx.x * (EMBED_THREADS >> a.log_g) + (threadIdx.x >> a.log_g);
    const int pack = first_pack + (threadIdx.x & (g - 1)), mine = packs - pack;  // (item i is there when i g < mine)
    const long long len = chunk_length(count, a.chunks), lo = chunk * len;
    const long long hi = lo + len < count ? lo + len : count;
    if (chunk >= a.chunks || mine <= 0 || lo >= hi) return;
    const T* dy = static_cast<const T*>(a.dy) + (long long)pack * V;
    d_table += (long long)pack * V;
    float* part = a.part + chunk * 2 * a.D + (long long)pack * V;
    const bool from_before = lo > 0 && a.keys[lo - 1] == a.keys[lo];
    const bool goes_on = hi < count && a.keys[hi] == a.keys[hi - 1];
    constexpr bool ASYNC = segment_async<T, V>;
    extern __shared__ __align__(16) unsigned char s_mem[];
    Pack<T, V>* ring = reinterpret_cast<Pack<T, V>*>(s_mem) + threadIdx.x;
    const auto slot = [&](int stage, int u, int i) { return ring + ((stage * CHUNK_STEP + u) * ITEMS + i) * EMBED_THREADS; };
    const auto source = [&](int place) { return reinterpret_cast<const Pack<T, V>*>(dy + (long long)place * a.D); };

    // Keys and places of a step (lo is a multiple of CHUNK_STEP and the sort's arrays are padded to 256
    // bytes: whole packs; what lies behind hi is not used).  Steps: positions lo + i CHUNK_STEP.
    const int length = (int)(hi - lo);
    const uint32_t* keys = a.keys + lo;
    const int* places = a.places + lo;
    Pack<int, 4> place[CHUNK_STEP / 4];  // of the next step to fetch
    const auto load_places = [&](int i) {
        if (i * CHUNK_STEP >= length) return;
#pragma unroll
        for (int q = 0; q < CHUNK_STEP / 4; ++q) place[q] = reinterpret_cast<const Pack<int, 4>*>(places + i * CHUNK_STEP)[q];
    };
    const auto fetch = [&](int i, int stage) {
        const int n = length - i * CHUNK_STEP;
#pragma unroll
        for (int u = 0; u < CHUNK_STEP; ++u) {
            if (u >= n) break;
            const Pack<T, V>* row = source(place[u / 4].v[u % 4]);
#pragma unroll
            for (int k = 0; k < ITEMS; ++k)
                if (k == 0 || k * g < mine) copy_async<sizeof(Pack<T, V>)>(slot(stage, u, k), row + k * g);
        }
    };

    // pipeline: step i is added while the rows of i + 1 and i + 2 are on their way and the places of
    // i + 3 are loaded
    static_assert(SEGMENT_STAGES == 3, "the pipeline below");
    load_places(0);
    if constexpr (ASYNC) {
        fetch(0, 0);
        copy_commit();
        load_places(1);
        fetch(1, 1);
        copy_commit();
        load_places(2);
    }
    uint32_t key = keys[0];
    bool first = true;
    Vals<V> sum[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) sum[i] = splat<V>(0.f);
    // the sum of the run that ends here: `crosses` when it goes on in the next chunk
    const auto finish_run = [&](bool crosses) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            if (i > 0 && i * g >= mine) break;
            if (first && from_before) reinterpret_cast<Pack<float, V>*>(part)[i * g] = to_pack<float, V>(sum[i]);
            else if (crosses) reinterpret_cast<Pack<float, V>*>(part + a.D)[i * g] = to_pack<float, V>(sum[i]);
            else store_pack<T, V>(d_table + (long long)key * a.D, i * g, sum[i], a.scale);
            sum[i] = splat<V>(0.f);
        }
        first = false;
    };
    int stage = 0;
    for (int i = 0; i * CHUNK_STEP < length; ++i) {
        const int n = length - i * CHUNK_STEP;
        Pack<uint32_t, 4> k[CHUNK_STEP / 4];
#pragma unroll
        for (int q = 0; q < CHUNK_STEP / 4; ++q) k[q] = reinterpret_cast<const Pack<uint32_t, 4>*>(keys + i * CHUNK_STEP)[q];
        Pack<T, V> v[CHUNK_STEP][ITEMS];
        if constexpr (ASYNC) {
            fetch(i + 2, stage == 0 ? 2 : stage - 1);
            copy_commit();
            load_places(i + 3);
            copy_wait<SEGMENT_STAGES - 1>();
        }
#pragma unroll
        for (int u = 0; u < CHUNK_STEP; ++u) {
            if (u >= n) break;
#pragma unroll
            for (int j = 0; j < ITEMS; ++j) {
                if (j > 0 && j * g >= mine) break;
                if constexpr (ASYNC) v[u][j] = *slot(stage, u, j);
                else v[u][j] = source(place[u / 4].v[u % 4])[j * g];
            }
        }
        if constexpr (!ASYNC) load_places(i + 1);
        stage = stage == 2 ? 0 : stage + 1;
#pragma unroll
        for (int u = 0; u < CHUNK_STEP; ++u) {
            if (u >= n) break;
            const uint32_t ku = k[u / 4].v[u % 4];
            if (ku != key) {  // (the same in every thread of the group)
                finish_run(false);
                key = ku;
            }
#pragma unroll
            for (int j = 0; j < ITEMS; ++j)
                if (j == 0 || j * g < mine) sum[j] = add(sum[j], to_vals<T, V>(v[u][j]));
        }
    }
    if constexpr (ASYNC) copy_wait<0>();
    finish_run(goes_on);
}

// Runs that cross chunk borders: the tail of the chunk in which the run starts, then the heads of
// the chunks that follow.  Q columns a thread.
//   Short runs, up to JOIN_SHORT heads: in the first blocks `span` threads (whole warps) per chunk that
//   may start one and slab of columns; a thread adds its columns up.
//   Longer ones (they contain a chunk whose number is a multiple of JOIN_SHORT): one block per such
//   chunk, which acts if it is the run's first.  32 threads across, 16 down: each of the 16 adds every
//   16th row, and the 16 sums are added in order.
// What bounds it is latency, a handful of dependent loads: 5 us behind the segments of 65536 places.
constexpr int JOIN_SHORT = 16;
constexpr int JOIN_THREADS = 512;
constexpr int JOIN_DOWN = JOIN_THREADS / 32;
template <typename T, int Q>
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(SegmentArgs a, int short_blocks, int short_slabs, int span) {
    __shared__ Pack<float, Q> s_sum[JOIN_DOWN][32];
    wait_for_previous();
    const int count = *a.count;
    const long long len = chunk_length(count, a.chunks);
    // whether chunk k exists and begins with the key / in the middle of a run of it
    const auto begins = [&](long long k, uint32_t key) { return k * len < count && a.keys[k * len] == key; };
    const auto continues = [&](long long k, uint32_t key) { return k > 0 && begins(k, key) && a.keys[k * len - 1] == key; };
    T* d_table = static_cast<T*>(a.d_table);
    const int lane = threadIdx.x & 31;
    const auto head = [&](long long k, long long c) {
        return to_vals<float, Q>(*reinterpret_cast<const Pack<float, Q>*>(a.part + k * 2 * a.D + c));
    };

    if ((int)blockIdx.x < short_blocks) {
        const long long unit = (long long)blockIdx.x * (JOIN_THREADS / span) + threadIdx.x / span;
        const long long k0 = unit / short_slabs;
        const long long c = ((unit % short_slabs) * span + threadIdx.x % span) * Q;
        if ((k0 + 1) * len >= count) return;  // (the same in a whole warp, like what follows)
        const uint32_t key = a.keys[(k0 + 1) * len];
        // lane i looks at chunk k0 + 1 + i: how many chunks in a row begin with the key
        static_assert(JOIN_SHORT < 32, "a warp looks past a short run");
        const unsigned going = ~__ballot_sync(0xffffffffu, begins(k0 + 1 + lane, key));
        const int heads = going ? __ffs(going) - 1 : 32;
        if (!continues(k0 + 1, key) || continues(k0, key)) return;  // nothing crosses, or it started before
        if (heads > JOIN_SHORT || c >= a.D) return;                 // a long one
        Vals<Q> sum = to_vals<float, Q>(*reinterpret_cast<const Pack<float, Q>*>(a.part + (k0 * 2 + 1) * a.D + c));
#pragma unroll 4
        for (int i = 0; i < heads; ++i) sum = add(sum, head(k0 + 1 + i, c));
        store_pack<T, Q>(d_table + (long long)key * a.D + c, 0, sum, a.scale);
        return;
    }

    const long long slabs = (a.D + 32 * Q - 1) / (32 * Q);
    const long long b = blockIdx.x - short_blocks;
    const long long m = (b / slabs + 1) * JOIN_SHORT;
    const int down = threadIdx.x >> 5;
    const long long c = ((b % slabs) * 32 + lane) * Q;
    if (m * len >= count) return;
    const uint32_t key = a.keys[m * len];
    // back to the chunk in which the run starts: lane i looks at chunk m - i
    const unsigned stops = ~__ballot_sync(0xffffffffu, continues(m - lane, key));
    const int back = stops ? __ffs(stops) - 1 : 32;
    if (back == 0 || back > JOIN_SHORT) return;  // nothing crosses here, or the run holds an earlier multiple
    const long long k0 = m - back;
    // on to the last chunk that begins with the key, 31 probes at a time: chunk `last` does, `end` does not
    long long last = m, end = a.chunks;
    while (end - last > 1) {
        const long long stride = (end - last + 31) / 32, at = last + (lane + 1) * stride;
        const unsigned over = ~__ballot_sync(0xffffffffu, at < end && begins(at, key));
        const int n = over ? __ffs(over) - 1 : 32;
        const long long next = last + (n + 1) * stride;
        last += n * stride;
        end = next < end ? next : end;
    }
    if (last - k0 <= JOIN_SHORT) return;  // a short one
    Vals<Q> sum = splat<Q>(0.f);
    if (c < a.D) {
#pragma unroll 8
        for (long long k = k0 + down; k <= last; k += JOIN_DOWN)
            sum = add(sum, to_vals<float, Q>(*reinterpret_cast<const Pack<float, Q>*>(a.part + (k * 2 + (k == k0)) * a.D + c)));
    }
    s_sum[down][lane] = to_pack<float, Q>(sum);
    __syncthreads();
    if (down || c >= a.D) return;
    for (int d = 1; d < JOIN_DOWN; ++d) sum = add(sum, to_vals<float, Q>(s_sum[d][lane]));
    store_pack<T, Q>(d_table + (long long)key * a.D + c, 0, sum, a.scale);
}

template <typename T, int V>
static void launch_sums(SegmentArgs& a, cudaStream_t s) {
    constexpr int Q = V < 4 ? V : 4;
    const long long packs = a.D / V;
    a.log_g = group_log((packs + segment_items<T, V> - 1) / segment_items<T, V>);
    const int groups = EMBED_THREADS >> a.log_g, slab = segment_items<T, V> << a.log_g;
    a.sum_blocks = (a.chunks + groups - 1) / groups;
    const long long zero = (a.rows + EMBED_THREADS - 1) / EMBED_THREADS;
    const dim3 grid((unsigned)(a.sum_blocks + (zero < 4096 ? zero : 4096)),
                    (unsigned)((packs + slab - 1) / slab));
    launch_chained(segment_kernel<T, V>, grid, EMBED_THREADS, segment_smem<T, V>, s, a);
    count_launch();
    int span = 32;
    while (span < JOIN_THREADS && span * Q < a.D) span *= 2;
    const long long short_slabs = (a.D + span * Q - 1) / (span * Q), long_slabs = (a.D + 32 * Q - 1) / (32 * Q);
    const long long short_blocks = ((a.chunks - 1) * short_slabs * span + JOIN_THREADS - 1) / JOIN_THREADS;
    const long long long_blocks = (a.chunks - 1) / JOIN_SHORT * long_slabs;
    if (a.chunks == 1) return;
    launch_chained(join_kernel<T, Q>, (unsigned)(short_blocks + long_blocks), JOIN_THREADS, 0, s, a, (int)short_blocks,
                   (int)short_slabs, span);
    count_launch();
}

// ---------------------------------------------------------------------------
// the call's plan and workspace: a pure function of the sizes and the device
// ---------------------------------------------------------------------------
struct EmbedPlan {
    int passes, bits, blocks, chunks;
    bool wide;  // one pass, the digit being the row
    size_t off_keys[2], off_places[2], off_hist, off_totals, off_count, off_part, bytes;
};

static int plan_embed_grad(long long n, long long rows, long long D, int dtype, int device, EmbedPlan* p) {
    if (n > EMBED_MAX_PLACES || rows > EMBED_MAX_ROWS || D > EMBED_MAX_WIDTH) return IGS_ERR_LIMIT;
    int bits = 1;
    while ((1ll << bits) < rows) ++bits;
    // (at most one sorting block an SM: they wait for each other, and all fit the device at once)
    const long long tiles = (n + SORT_BLOCK - 1) / SORT_BLOCK;
    p->blocks = (int)(tiles < sm_count(device) ? tiles : sm_count(device));
    p->wide = bits > SORT_MAX_BITS && bits <= WIDE_MAX_BITS && tiles == p->blocks;
    p->passes = p->wide ? 1 : (bits + SORT_MAX_BITS - 1) / SORT_MAX_BITS;
    p->bits = (bits + p->passes - 1) / p->passes;
    // One wave of blocks: 512 threads an SM, 16 bytes of columns a thread.
    const long long packs = (D * (long long)dtype_size(dtype) + 15) / 16, g = 1ll << group_log(packs);
    long long chunks = (long long)sm_count(device) * 512 / ((packs + g - 1) / g * g);
    if (chunks < sm_count(device) / 2) chunks = sm_count(device) / 2;
    if (chunks > (n + CHUNK_STEP - 1) / CHUNK_STEP) chunks = (n + CHUNK_STEP - 1) / CHUNK_STEP;
    p->chunks = (int)(chunks < 1 ? 1 : chunks);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t r = at;
        at += align_up(bytes, 256);
        return r;
    };
    for (int i = 0; i < 2; ++i) {
        p->off_keys[i] = take((size_t)n * 4);
        p->off_places[i] = take((size_t)n * 4);
    }
    p->off_hist = take((size_t)(1 << p->bits) * p->blocks * 4);
    p->off_totals = take(((size_t)(1 << p->bits) + (1 << WIDE_MAX_BITS) / SORT_THREADS) * 4);
    p->off_count = take(4);
    p->off_part = take((size_t)p->chunks * 2 * D * 4);
    p->bytes = at;
    return IGS_OK;
}

// A cooperative launch of sorting blocks.
static cudaError_t launch_waiting(void (*kernel)(SortArgs), size_t smem, SortArgs& a, int blocks, int device,
                                  cudaStream_t s) {
    static bool attr_set[64] = {};
    if (smem > 48 * 1024 && (device < 0 || device >= 64 || !attr_set[device])) {
        const cudaError_t e = cudaFuncSetAttribute(sort_wide_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   (int)(sizeof(unsigned) << WIDE_MAX_BITS));
        if (e != cudaSuccess) return e;
        if (device >= 0 && device < 64) attr_set[device] = true;
    }
    void* args[] = {&a};
    return cudaLaunchCooperativeKernel(reinterpret_cast<const void*>(kernel), dim3((unsigned)blocks), dim3(SORT_THREADS), args,
                                       smem, s);
}

static int token_args_ok(int token_bytes, long long n, long long rows, long long D, int dtype, float scale) {
    if ((token_bytes != 4 && token_bytes != 8) || n < 0 || rows < 1 || D < 1 || !dtype_ok(dtype)) return IGS_ERR_ARG;
    if (!(scale - scale == 0.f)) return IGS_ERR_ARG;  // a finite number
    if (n > EMBED_MAX_PLACES || rows > EMBED_MAX_ROWS || D > EMBED_MAX_WIDTH) return IGS_ERR_LIMIT;
    return IGS_OK;
}

}  // namespace igs

using namespace igs;

extern "C" int igs_embed(const void* tokens, int token_bytes, long long n, const void* table, int dtype, long long rows,
                         long long D, long long row_stride, float scale, int has_empty, long long empty, void* out,
                         int device, void* stream) {
    const int rc = token_args_ok(token_bytes, n, rows, D, dtype, scale);
    if (rc) return rc;
    if (row_stride < 0) return IGS_ERR_ARG;
    if (n == 0) return IGS_OK;
    if (!tokens || !table || !out) return IGS_ERR_ARG;
    DeviceGuard guard(device);
    if (!guard.ok) return IGS_ERR_DEVICE;
    cudaStream_t s = (cudaStream_t)stream;
    EmbedArgs a{{tokens, token_bytes == 8, has_empty != 0, empty, rows}, table, out, n, D, row_stride, scale};
    const int bytes = embed_pack_bytes(table, out, D, row_stride, dtype_size(dtype));
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        if (bytes == 16) launch_embed<T, 16 / sizeof(T)>(a, device, s);
        else if (bytes == 4) launch_embed<T, 4 / sizeof(T)>(a, device, s);
        else launch_embed<T, 1>(a, device, s);
        return 0;
    });
    count_launch();
    return (int)cudaGetLastError();
}

extern "C" int igs_embed_grad_workspace_bytes(long long n, long long rows, long long D, int dtype, int device,
                                              size_t* bytes) {
    if (n < 0 || rows < 1 || D < 1 || !dtype_ok(dtype) || !bytes) return IGS_ERR_ARG;
    EmbedPlan p;
    const int rc = plan_embed_grad(n, rows, D, dtype, device, &p);
    if (rc) return rc;
    *bytes = p.bytes;
    return IGS_OK;
}

extern "C" int igs_embed_grad(const void* tokens, int token_bytes, long long n, const void* dy, int dtype,
                              long long rows, long long D, float scale, int has_empty, long long empty, void* d_table,
                              void* workspace, size_t workspace_bytes, int device, void* stream) {
    int rc = token_args_ok(token_bytes, n, rows, D, dtype, scale);
    if (rc) return rc;
    if (!d_table || (n > 0 && (!tokens || !dy))) return IGS_ERR_ARG;
    EmbedPlan p;
    rc = plan_embed_grad(n, rows, D, dtype, device, &p);
    if (rc) return rc;
    if (n > 0 && (!workspace || workspace_bytes < p.bytes || !aligned_to(workspace, 16))) return IGS_ERR_WORKSPACE;
    DeviceGuard guard(device);
    if (!guard.ok) return IGS_ERR_DEVICE;
    cudaStream_t s = (cudaStream_t)stream;
    if (n == 0) return (int)cudaMemsetAsync(d_table, 0, (size_t)rows * D * dtype_size(dtype), s);

    unsigned char* ws = static_cast<unsigned char*>(workspace);
    SortArgs so{};
    so.tokens = Tokens{tokens, token_bytes == 8, has_empty != 0, empty, rows};
    for (int i = 0; i < 2; ++i) {
        so.keys[i] = reinterpret_cast<uint32_t*>(ws + p.off_keys[i]);
        so.places[i] = reinterpret_cast<int*>(ws + p.off_places[i]);
    }
    so.hist = reinterpret_cast<int*>(ws + p.off_hist);
    so.totals = reinterpret_cast<int*>(ws + p.off_totals);
    so.count = reinterpret_cast<int*>(ws + p.off_count);
    so.n = n;
    so.passes = p.passes;
    so.bits = p.bits;
    int sorted = 0;
    if (n <= RANK_MAX) {
        sort_rank_kernel<<<(unsigned)((n + 31) / 32), RANK_WARPS * 32, 0, s>>>(so);
    } else {
        const cudaError_t e = p.wide ? launch_waiting(sort_wide_kernel, sizeof(unsigned) << p.bits, so, p.blocks, device, s)
                                     : launch_waiting(sort_kernel, 0, so, p.blocks, device, s);
        if (e != cudaSuccess) {
            cudaGetLastError();
            return (int)e;
        }
        sorted = (p.passes & 1) ^ 1;
    }
    count_launch();
    SegmentArgs a{so.keys[sorted], so.places[sorted], so.count, dy, d_table, reinterpret_cast<float*>(ws + p.off_part), rows, D,
                  scale, p.chunks, 0, 0};
    const int bytes = embed_pack_bytes(dy, d_table, D, D, dtype_size(dtype));
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        if (bytes == 16) launch_sums<T, 16 / sizeof(T)>(a, s);
        else if (bytes == 4) launch_sums<T, 4 / sizeof(T)>(a, s);
        else launch_sums<T, 1>(a, s);
        return 0;
    });
    return (int)cudaGetLastError();
}
