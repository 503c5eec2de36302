// igs_embed: rows of a table by token, times a scale.  igs_embed_grad: the table's gradient,
//   d_table[v] = scale * sum of dy[i] over the places i with tokens[i] == v,
// dense, zeros for rows without a token.
//
// The gradient goes by sorted tokens instead of atomics: a stable sort of (token, place) puts the
// places of one token next to each other in their own order, so every row is one sum in 32 bits
// with a fixed sequence and one rounding, the same bits on every run.
//   1. sort: least significant digits first, up to 10 bits a pass (a codebook of a million rows
//      needs two); per pass a count per block of places, a prefix sum over blocks, and the
//      placement.  Places without a token in the table drop out in the first pass.
//   2. segments: the sorted places are cut into chunks of equal length whatever the tokens are
//      (one common token may own most of them).  A run of one token inside a chunk is finished
//      there; the sums of runs that cross a border go to the chunk's two partial rows ("head":
//      it came from the chunk before, "tail": it started here and goes on).  The same launch
//      writes the zero rows.
//   3. join: the chunk in which a crossing run started adds the run's partial rows in order.
#include "feature.cuh"

namespace igs {

constexpr int EMBED_THREADS = 128;
constexpr int SORT_THREADS = 256;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int SORT_PER_WARP = 256;                       // places a warp ranks, 32 at a time
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

// one CTA per place (and on): a row of D values
template <typename T>
__global__ void __launch_bounds__(EMBED_THREADS) embed_kernel(EmbedArgs a) {
    for (long long i = blockIdx.x; i < a.n; i += gridDim.x) {
        const long long tok = token_at(a.tokens, i);
        const uint32_t row = row_of(a.tokens, tok);
        T* out = static_cast<T*>(a.out) + i * a.D;
        if (row != NO_ROW) {
            const T* src = static_cast<const T*>(a.table) + (long long)row * a.row_stride;
            for (long long c = threadIdx.x; c < a.D; c += EMBED_THREADS) out[c] = from_f<T>(to_f(src[c]) * a.scale);
        } else {
            // an empty place is zero; a token outside the table is an error that shows: NaN
            const bool empty = a.tokens.has_empty && tok == a.tokens.empty;
            const T v = from_f<T>(empty ? 0.f : __int_as_float(0x7fc00000));
            for (long long c = threadIdx.x; c < a.D; c += EMBED_THREADS) out[c] = v;
        }
    }
}

// ---------------------------------------------------------------------------
// sort
// ---------------------------------------------------------------------------
struct SortArgs {
    Tokens tokens;
    const uint32_t* keys_in;   // NULL in the first pass: the tokens themselves
    const int* places_in;
    uint32_t* keys_out;
    int* places_out;
    int* hist;                 // [digits][blocks]: counts, then first slots within the digit
    int* totals;               // [digits]
    const int* count_in;       // how many (key, place) pairs the pass takes; first pass: n
    int* count_out;            // first pass: how many places hold a token
    long long n;
    int n_blocks, shift, digits;
};

// the pair at position i of the pass's input; false when there is none
__device__ __forceinline__ bool sort_load(const SortArgs& a, long long i, long long count, uint32_t& key, int& place) {
    if (i >= count) return false;
    if (a.keys_in) {
        key = a.keys_in[i];
        place = a.places_in[i];
        return true;
    }
    key = row_of(a.tokens, token_at(a.tokens, i));
    place = (int)i;
    return key != NO_ROW;
}

__global__ void __launch_bounds__(SORT_THREADS) sort_count_kernel(SortArgs a) {
    __shared__ int s_hist[SORT_MAX_DIGITS];
    for (int d = threadIdx.x; d < a.digits; d += SORT_THREADS) s_hist[d] = 0;
    __syncthreads();
    const long long count = a.keys_in ? *a.count_in : a.n;
    const long long base = (long long)blockIdx.x * SORT_BLOCK;
    for (int j = threadIdx.x; j < SORT_BLOCK; j += SORT_THREADS) {
        uint32_t key;
        int place;
        // (integer counts: the result does not depend on the order of the adds)
        if (sort_load(a, base + j, count, key, place)) atomicAdd(&s_hist[(key >> a.shift) & (a.digits - 1)], 1);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < a.digits; d += SORT_THREADS) a.hist[(long long)d * a.n_blocks + blockIdx.x] = s_hist[d];
}

// a warp per digit: exclusive prefix sums over the blocks, and the digit's total
__global__ void __launch_bounds__(SORT_THREADS) sort_scan_kernel(SortArgs a) {
    const int d = blockIdx.x * SORT_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (d >= a.digits) return;
    int* h = a.hist + (long long)d * a.n_blocks;
    int run = 0;
    for (int b0 = 0; b0 < a.n_blocks; b0 += 32) {
        const int b = b0 + lane;
        const int v = b < a.n_blocks ? h[b] : 0;
        int incl = v;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, incl, s);
            if (lane >= s) incl += t;
        }
        if (b < a.n_blocks) h[b] = run + incl - v;
        run += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) a.totals[d] = run;
}

// places of a block in order: warp w takes SORT_PER_WARP neighbours, 32 at a time
__global__ void __launch_bounds__(SORT_THREADS) sort_place_kernel(SortArgs a) {
    __shared__ int s_first[SORT_MAX_DIGITS];              // the block's first slot per digit
    __shared__ int s_warp[SORT_WARPS][SORT_MAX_DIGITS];   // per warp: counts, then first slots
    __shared__ int s_sum[SORT_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

    // first slot of every digit: exclusive sums of the totals, four digits a thread
    constexpr int PER = SORT_MAX_DIGITS / SORT_THREADS;
    int t[PER], sum = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int d = threadIdx.x * PER + j;
        t[j] = d < a.digits ? a.totals[d] : 0;
        sum += t[j];
    }
    int incl = sum;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, s);
        if (lane >= s) incl += v;
    }
    if (lane == 31) s_sum[warp] = incl;
    for (int d = threadIdx.x; d < SORT_WARPS * SORT_MAX_DIGITS; d += SORT_THREADS) (&s_warp[0][0])[d] = 0;
    __syncthreads();
    int run = incl - sum;
    for (int w = 0; w < warp; ++w) run += s_sum[w];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int d = threadIdx.x * PER + j;
        if (d < a.digits) s_first[d] = run + a.hist[(long long)d * a.n_blocks + blockIdx.x];
        run += t[j];
    }
    if (a.count_out && blockIdx.x == 0 && threadIdx.x == SORT_THREADS - 1) *a.count_out = run;

    // rank within the warp, in order of place
    const long long count = a.keys_in ? *a.count_in : a.n;
    const long long base = (long long)blockIdx.x * SORT_BLOCK + (long long)warp * SORT_PER_WARP;
    uint32_t key[SORT_PER_WARP / 32];
    int place[SORT_PER_WARP / 32], rank[SORT_PER_WARP / 32];
#pragma unroll
    for (int j = 0; j < SORT_PER_WARP / 32; ++j) {
        const bool ok = sort_load(a, base + j * 32 + lane, count, key[j], place[j]);
        if (!ok) key[j] = NO_ROW;
        // pairs that are not there share a digit no pair has, so they match only each other
        const int d = ok ? (int)((key[j] >> a.shift) & (a.digits - 1)) : SORT_MAX_DIGITS;
        const unsigned peers = __match_any_sync(0xffffffffu, d);
        const int before = __popc(peers & ((1u << lane) - 1u));
        rank[j] = ok ? s_warp[warp][d] + before : 0;
        __syncwarp();
        if (ok && before == 0) s_warp[warp][d] += __popc(peers);
        __syncwarp();
    }
    __syncthreads();
    for (int d = threadIdx.x; d < a.digits; d += SORT_THREADS) {
        int slot = s_first[d];
#pragma unroll
        for (int w = 0; w < SORT_WARPS; ++w) {
            const int c = s_warp[w][d];
            s_warp[w][d] = slot;
            slot += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SORT_PER_WARP / 32; ++j) {
        if (key[j] == NO_ROW) continue;
        const long long slot = s_warp[warp][(key[j] >> a.shift) & (a.digits - 1)] + rank[j];
        // slot < n by construction; the guard keeps a corrupted workspace from turning into a stray write
        if (slot >= 0 && slot < a.n) {
            a.keys_out[slot] = key[j];
            a.places_out[slot] = place[j];
        }
    }
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
    int sum_blocks, zero_blocks;
};

// positions [lo, hi) of a chunk
__device__ __forceinline__ long long chunk_length(long long count, int chunks) { return (count + chunks - 1) / chunks; }

// whether a row has a token: binary search
__device__ __forceinline__ bool has_key(const uint32_t* keys, int count, uint32_t row) {
    int lo = 0, hi = count;
    while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        if (keys[mid] < row) lo = mid + 1; else hi = mid;
    }
    return lo < count && keys[lo] == row;
}

// grid (sum blocks + zero blocks, column slabs).  Sum blocks: one chunk each, one column a thread.
template <typename T>
__global__ void __launch_bounds__(EMBED_THREADS) segment_kernel(SegmentArgs a) {
    const int count = *a.count;
    T* d_table = static_cast<T*>(a.d_table);
    const long long c = (long long)blockIdx.y * EMBED_THREADS + threadIdx.x;
    if ((int)blockIdx.x >= a.sum_blocks) {
        // rows without a token
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        const long long group = (long long)(blockIdx.x - a.sum_blocks) * (EMBED_THREADS / 32) + warp;
        const long long groups = (long long)a.zero_blocks * (EMBED_THREADS / 32);
        if (blockIdx.y) return;
        for (long long r0 = group * 32; r0 < a.rows; r0 += groups * 32) {
            const long long r = r0 + lane;
            unsigned absent = __ballot_sync(0xffffffffu, r < a.rows && !has_key(a.keys, count, (uint32_t)r));
            while (absent) {
                const int k = __ffs(absent) - 1;
                absent &= absent - 1;
                for (long long i = lane; i < a.D; i += 32) d_table[(r0 + k) * a.D + i] = from_f<T>(0.f);
            }
        }
        return;
    }
    if (c >= a.D) return;
    const long long len = chunk_length(count, a.chunks), lo = blockIdx.x * len;
    const long long hi = lo + len < count ? lo + len : count;
    if (lo >= hi) return;
    const T* dy = static_cast<const T*>(a.dy);
    const bool from_before = lo > 0 && a.keys[lo - 1] == a.keys[lo];
    const bool goes_on = hi < count && a.keys[hi] == a.keys[hi - 1];
    float* part = a.part + (long long)blockIdx.x * 2 * a.D;
    uint32_t key = a.keys[lo];
    bool first = true;
    float sum = 0.f;
    for (long long p = lo; p < hi; ++p) {
        const uint32_t k = a.keys[p];
        if (k != key) {
            if (first && from_before)
                part[c] = sum;
            else
                d_table[(long long)key * a.D + c] = from_f<T>(sum * a.scale);
            first = false;
            key = k;
            sum = 0.f;
        }
        sum += to_f(dy[(long long)a.places[p] * a.D + c]);
    }
    if (first && from_before)
        part[c] = sum;
    else if (goes_on)
        part[a.D + c] = sum;
    else
        d_table[(long long)key * a.D + c] = from_f<T>(sum * a.scale);
}

// grid (chunks, column slabs): the chunk in which a crossing run starts adds the run up
template <typename T>
__global__ void __launch_bounds__(EMBED_THREADS) join_kernel(SegmentArgs a) {
    const int count = *a.count;
    const long long len = chunk_length(count, a.chunks), lo = blockIdx.x * len, hi = lo + len;
    const long long c = (long long)blockIdx.y * EMBED_THREADS + threadIdx.x;
    if (c >= a.D || hi >= count) return;
    const uint32_t key = a.keys[hi - 1];
    if (a.keys[hi] != key) return;                                          // nothing crosses the border
    if (lo > 0 && a.keys[lo] == key && a.keys[lo - 1] == key) return;       // it started further to the left
    float sum = a.part[(long long)blockIdx.x * 2 * a.D + a.D + c];
    for (long long k = blockIdx.x + 1; k * len < count && a.keys[k * len] == key; ++k) sum += a.part[k * 2 * a.D + c];
    static_cast<T*>(a.d_table)[(long long)key * a.D + c] = from_f<T>(sum * a.scale);
}

// ---------------------------------------------------------------------------
// the call's plan and workspace: a pure function of the sizes and the device
// ---------------------------------------------------------------------------
struct EmbedPlan {
    int passes, bits, n_blocks, chunks;
    size_t off_keys[2], off_places[2], off_hist, off_totals, off_count, off_part, bytes;
};

static int plan_embed_grad(long long n, long long rows, long long D, int device, EmbedPlan* p) {
    if (n > EMBED_MAX_PLACES || rows > EMBED_MAX_ROWS || D > EMBED_MAX_WIDTH) return IGS_ERR_LIMIT;
    int bits = 1;
    while ((1ll << bits) < rows) ++bits;
    p->passes = (bits + SORT_MAX_BITS - 1) / SORT_MAX_BITS;
    p->bits = (bits + p->passes - 1) / p->passes;
    p->n_blocks = (int)((n + SORT_BLOCK - 1) / SORT_BLOCK);
    // enough chunks to fill the device once the column slabs are counted, none shorter than 16 places
    const long long slabs = (D + EMBED_THREADS - 1) / EMBED_THREADS;
    long long chunks = (long long)sm_count(device) * 16 / slabs;
    if (chunks > (n + 15) / 16) chunks = (n + 15) / 16;
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
    p->off_hist = take((size_t)(1 << p->bits) * p->n_blocks * 4);
    p->off_totals = take((size_t)(1 << p->bits) * 4);
    p->off_count = take(4);
    p->off_part = take((size_t)p->chunks * 2 * D * 4);
    p->bytes = at;
    return IGS_OK;
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
    with_dtype(dtype, [&](auto t) {
        embed_kernel<decltype(t)><<<(unsigned)n, EMBED_THREADS, 0, s>>>(a);
        return 0;
    });
    count_launch();
    return (int)cudaGetLastError();
}

extern "C" int igs_embed_grad_workspace_bytes(long long n, long long rows, long long D, int device, size_t* bytes) {
    if (n < 0 || rows < 1 || D < 1 || !bytes) return IGS_ERR_ARG;
    EmbedPlan p;
    const int rc = plan_embed_grad(n, rows, D, device, &p);
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
    rc = plan_embed_grad(n, rows, D, device, &p);
    if (rc) return rc;
    if (n > 0 && (!workspace || workspace_bytes < p.bytes)) return IGS_ERR_WORKSPACE;
    DeviceGuard guard(device);
    if (!guard.ok) return IGS_ERR_DEVICE;
    cudaStream_t s = (cudaStream_t)stream;
    if (n == 0) return (int)cudaMemsetAsync(d_table, 0, (size_t)rows * D * dtype_size(dtype), s);

    unsigned char* ws = static_cast<unsigned char*>(workspace);
    SortArgs so{};
    so.tokens = Tokens{tokens, token_bytes == 8, has_empty != 0, empty, rows};
    so.hist = reinterpret_cast<int*>(ws + p.off_hist);
    so.totals = reinterpret_cast<int*>(ws + p.off_totals);
    int* count = reinterpret_cast<int*>(ws + p.off_count);
    so.count_in = count;
    so.n = n;
    so.n_blocks = p.n_blocks;
    so.digits = 1 << p.bits;
    for (int pass = 0; pass < p.passes; ++pass) {
        const int to = pass & 1;
        so.keys_in = pass ? reinterpret_cast<uint32_t*>(ws + p.off_keys[to ^ 1]) : nullptr;
        so.places_in = pass ? reinterpret_cast<int*>(ws + p.off_places[to ^ 1]) : nullptr;
        so.keys_out = reinterpret_cast<uint32_t*>(ws + p.off_keys[to]);
        so.places_out = reinterpret_cast<int*>(ws + p.off_places[to]);
        so.count_out = pass ? nullptr : count;
        so.shift = pass * p.bits;
        sort_count_kernel<<<p.n_blocks, SORT_THREADS, 0, s>>>(so);
        sort_scan_kernel<<<(so.digits + SORT_WARPS - 1) / SORT_WARPS, SORT_THREADS, 0, s>>>(so);
        sort_place_kernel<<<p.n_blocks, SORT_THREADS, 0, s>>>(so);
        count_launch(3);
    }
    SegmentArgs a{so.keys_out, so.places_out, count, dy, d_table, reinterpret_cast<float*>(ws + p.off_part), rows, D,
                  scale, p.chunks, p.chunks, 0};
    const long long zero = (rows + EMBED_THREADS - 1) / EMBED_THREADS;
    a.zero_blocks = (int)(zero < 4096 ? zero : 4096);
    const unsigned slabs = (unsigned)((D + EMBED_THREADS - 1) / EMBED_THREADS);
    with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        segment_kernel<T><<<dim3((unsigned)(a.sum_blocks + a.zero_blocks), slabs), EMBED_THREADS, 0, s>>>(a);
        if (a.chunks > 1) join_kernel<T><<<dim3((unsigned)a.chunks, slabs), EMBED_THREADS, 0, s>>>(a);
        return 0;
    });
    count_launch(a.chunks > 1 ? 2 : 1);
    return (int)cudaGetLastError();
}
