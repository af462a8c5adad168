// k_kvcache_q8.cu -- KV cache held as int8 codes: quantised as it is written,
// and read back.
//
// Caches [batch, kv_heads, max_seq, head_dim] int8 with f32 scales [batch,
// kv_heads, nblk], one for each block of `block` consecutive positions of a
// head (nblk = ceil(max_seq / block)); a code c stands for c * scale.  The
// unquantised append is KVCache::update (src/cache/kv_cache.rs:55-85); the
// 8-bit form has no counterpart in the reference.
//
// Append.  A block that receives tokens needs the scale need = max|x| / 127
// over the tokens it receives.  If it holds no token of its sequence yet (it
// starts at or behind the sequence's cached length) its scale becomes need;
// otherwise max(old, need), and where that is larger than the old scale the
// codes of the tokens it holds are restated, c' = nearest(c old / new) -- at
// most one more rounding of half a step each time the scale grows, and none
// for blocks written whole.  c' depends on |c| only, so the 128 quotients are
// computed once into a table and the codes looked up.
//
// Layout.  An item is one touched block of one head of k or v: its new tokens
// are one contiguous run in the source and in the cache, so a warp (runs of
// at most 128 16-byte vectors) or a CTA loads the run once into registers,
// reduces, and writes the codes: each byte crosses HBM once.  Bound by HBM
// bytes and by instructions alike for prompts (8 of up to 2048 tokens, 8 heads x
// 128, bf16, k and v: 18.7 us, 4.0 TB/s of 3 bytes an element, 62 % of the issue
// slots, half of them on the integer pipe), by launch latency for single tokens
// (64 sequences 2.6 us).
//
// Read back is one pass, x = c * scale rounded to the output type (8 sequences of
// up to 8192 keys, 8 heads x 128, bf16: 62.8 us, 5.3 TB/s).
#include "oxide_q8.cuh"

namespace oxide {

struct AppendQ8Args {
    const int32_t* cur_lens;   // per sequence; NULL: cur_len
    const int32_t* new_lens;   // per sequence; NULL: new_len
    uint32_t max_seq, cur_len, new_len;
    uint32_t head_dim, nblk, shift;  // block = 1 << shift
    uint32_t half;             // heads * wide: items of k; as many of v follow
    uint32_t items;            // 2 * half
    FastDiv wide, kv_heads;    // wide: blocks an append can touch
};

// One item: the block, the positions [lo, hi) it receives, where they come
// from and go to (positions are below 2^31).
struct AppendItem {
    bool is_v;
    bool holds;               // tokens of this sequence before lo are in the block
    uint32_t bh, blk;
    uint32_t lo, hi, start;   // new positions; the block's first position
    uint64_t src;             // first new row in k / v, counted in rows
};
__device__ __forceinline__ bool append_item(const AppendQ8Args& p, uint32_t i, AppendItem& it) {
    it.is_v = i >= p.half;
    const uint32_t r = it.is_v ? i - p.half : i;
    it.bh = p.wide.div(r);
    const uint32_t j = r - it.bh * p.wide.d;
    uint32_t cur = p.cur_len, n = p.new_len;
    if (p.cur_lens || p.new_lens) {
        const uint32_t b = p.kv_heads.div(it.bh);
        if (p.cur_lens) {
            cur = (uint32_t)__ldg(p.cur_lens + b);
            if (cur > p.max_seq) return false;  // negative ones too
        }
        if (p.new_lens) {
            const int32_t c = __ldg(p.new_lens + b);
            n = c <= 0 ? 0u : min((uint32_t)c, n);
        }
    }
    if (n == 0 || n > p.max_seq - cur) return false;  // nothing to write, or it does not fit: the sequence is left as it is
    it.blk = (cur >> p.shift) + j;
    if (it.blk >= p.nblk) return false;
    it.start = it.blk << p.shift;
    const uint32_t end = cur + n;
    if (it.start >= end) return false;
    it.lo = max(it.start, cur);
    it.hi = min(it.start + (1u << p.shift), end);
    it.src = (uint64_t)it.bh * p.new_len + (it.lo - cur);
    it.holds = it.start < cur;
    return true;
}

// The block's scale after this append, whether it is the new tokens' own, and
// whether the codes the block holds are restated.
// Scales are compared as bits, which carries a NaN along.
__device__ __forceinline__ float append_scale(const AppendItem& it, float had, uint32_t amax, bool& fresh, bool& grown) {
    const float need = q8_scale_of(amax);
    fresh = true;
    grown = false;
    if (!it.holds) return need;
    const uint32_t a = q8_abs_bits(had), b = q8_abs_bits(need);
    fresh = b > a;
    grown = fresh && b < Q8_INF;
    return fresh ? need : __uint_as_float(a);
}

// Restate the codes of positions [start, lo) from scale `had` to scale `s`.
// `lut` (128 bytes of shared memory) is this group's own; TPI threads take part.
template <int TPI>
__device__ __forceinline__ void append_restate(int8_t* head, const AppendQ8Args& p, const AppendItem& it, float had,
                                               float s, uint8_t* lut, uint32_t t) {
    for (uint32_t i = t; i < 128; i += TPI) lut[i] = (uint8_t)q8_restated((int)i, had, s);
    if (TPI == 32) __syncwarp();
    else __syncthreads();
    int8_t* c = head + (uint64_t)it.start * p.head_dim;
    const uint32_t n = (it.lo - it.start) * p.head_dim;
    auto restate = [&](int v) -> uint32_t {
        const int a = v < 0 ? (v < -127 ? 127 : -v) : v;
        const int q = lut[a];
        return (uint32_t)(v < 0 ? -q : q) & 0xffu;
    };
    if (p.head_dim % 4 == 0 && (reinterpret_cast<uintptr_t>(c) & 3) == 0) {
        uint32_t* w = reinterpret_cast<uint32_t*>(c);
#pragma unroll 4
        for (uint32_t i = t; i < n / 4; i += TPI) {
            const uint32_t v = w[i];
            w[i] = restate((int8_t)v) | restate((int8_t)(v >> 8)) << 8 | restate((int8_t)(v >> 16)) << 16 |
                   restate((int8_t)(v >> 24)) << 24;
        }
    } else {
        for (uint32_t i = t; i < n; i += TPI) c[i] = (int8_t)restate(c[i]);
    }
}

// Largest |x| bits over the group's threads (contains __syncthreads() for a CTA).
template <int TPI>
__device__ __forceinline__ uint32_t append_max(uint32_t a) {
    a = q8_warp_max(a);
    if (TPI == 32) return a;
    __shared__ uint32_t red[32];
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = a;
    __syncthreads();
    a = red[0];
#pragma unroll
    for (int i = 1; i < TPI / 32; ++i) a = max(a, red[i]);
    __syncthreads();
    return a;
}

// TPI threads an item (32: eight items per CTA), VPT vectors a thread.
template <typename T, int TPI, int VPT>
__global__ void __launch_bounds__(TPI == 32 ? 256 : TPI, TPI == 256 ? 4 : 1)
    kv_append_q8_vec_kernel(int8_t* kc, int8_t* vc, float* ks, float* vs, const T* k, const T* v, AppendQ8Args p) {
    pdl_begin();
    constexpr int V = Vec<T>::N, IPC = TPI == 32 ? 8 : 1;
    __shared__ uint8_t luts[IPC][128];
    const uint32_t t = TPI == 32 ? threadIdx.x & 31 : threadIdx.x, g = TPI == 32 ? threadIdx.x >> 5 : 0;
    for (uint64_t i = (uint64_t)blockIdx.x * IPC + g; i < p.items; i += (uint64_t)gridDim.x * IPC) {
        AppendItem it;
        if (!append_item(p, (uint32_t)i, it)) continue;  // the same for the whole group
        const T* src = (it.is_v ? v : k) + it.src * p.head_dim;
        int8_t* head = (it.is_v ? vc : kc) + (uint64_t)it.bh * p.max_seq * p.head_dim;
        float* sp = (it.is_v ? vs : ks) + (uint64_t)it.bh * p.nblk + it.blk;
        const uint32_t nvec = (it.hi - it.lo) * p.head_dim / V;
        uint4 raw[VPT];
#pragma unroll
        for (int u = 0; u < VPT; ++u)
            if (t + u * TPI < nvec) raw[u] = ld_stream(src + (uint64_t)(t + u * TPI) * V);
        const float had = it.holds ? *reinterpret_cast<volatile float*>(sp) : 0.0f;
        uint32_t a = 0;
#pragma unroll
        for (int u = 0; u < VPT; ++u)
            if (t + u * TPI < nvec) a = q8_vec_amax(raw[u], a, T());
        a = append_max<TPI>(q8_amax_join(a, T()));  // also: every thread has read the old scale
        bool fresh, grown;
        const float s = append_scale(it, had, a, fresh, grown);
        if (t == 0) *sp = s;
        const Q8Coder<T> coder(s, fresh ? __uint_as_float(a) : -1.0f);
        int8_t* dst = head + (uint64_t)it.lo * p.head_dim;
        uint32_t open = 0;  // vectors with codes that the definition has to decide
#pragma unroll
        for (int u = 0; u < VPT; ++u)
            if (t + u * TPI < nvec) {
                float x[V];
                uint32_t c[V / 4];
                Vec<T>::unpack(raw[u], x);
                open |= (q8_codes<V>(coder, x, c) ? 1u : 0u) << u;
                q8_store(dst + (t + u * TPI) * V, c);
            }
        if (open) {  // once more, behind the other stores: a branch at every vector kept them from overlapping
#pragma unroll
            for (int u = 0; u < VPT; ++u)
                if (open >> u & 1u) {
                    uint32_t c[V / 4];
                    q8_take(c, q8_decide<T>(raw[u], s));
                    q8_store(dst + (t + u * TPI) * V, c);
                }
        }
        if (grown) {
            append_restate<TPI>(head, p, it, had, s, luts[g], t);
            if (TPI == 32) __syncwarp();  // the table is written again for the next item
            else __syncthreads();
        }
    }
}

// Any head size and alignment: the run is read twice.
template <typename T, int TPI>
__global__ void __launch_bounds__(256)
    kv_append_q8_scalar_kernel(int8_t* kc, int8_t* vc, float* ks, float* vs, const T* k, const T* v, AppendQ8Args p) {
    pdl_begin();
    constexpr int IPC = 256 / TPI;
    __shared__ uint8_t luts[IPC][128];
    const uint32_t t = threadIdx.x % TPI, g = threadIdx.x / TPI;
    for (uint64_t i = (uint64_t)blockIdx.x * IPC + g; i < p.items; i += (uint64_t)gridDim.x * IPC) {
        AppendItem it;
        if (!append_item(p, (uint32_t)i, it)) continue;
        const T* src = (it.is_v ? v : k) + it.src * p.head_dim;
        int8_t* head = (it.is_v ? vc : kc) + (uint64_t)it.bh * p.max_seq * p.head_dim;
        float* sp = (it.is_v ? vs : ks) + (uint64_t)it.bh * p.nblk + it.blk;
        const uint32_t n = (it.hi - it.lo) * p.head_dim;
        const float had = it.holds ? *reinterpret_cast<volatile float*>(sp) : 0.0f;
        uint32_t a = 0;
        for (uint32_t e = t; e < n; e += TPI) a = max(a, q8_abs_bits(Vec<T>::load1(src + e)));
        a = append_max<TPI>(a);
        bool fresh, grown;
        const float s = append_scale(it, had, a, fresh, grown);
        if (t == 0) *sp = s;
        const Q8Coder<T> coder(s, fresh ? __uint_as_float(a) : -1.0f);
        int8_t* dst = head + (uint64_t)it.lo * p.head_dim;
        for (uint32_t e = t; e < n; e += TPI) {
            const float x = Vec<T>::load1(src + e);
            dst[e] = (int8_t)q8_code(coder, x, [&] { return q8_definition(x, s); });
        }
        if (grown) {
            append_restate<TPI>(head, p, it, had, s, luts[g], t);
            if (TPI == 32) __syncwarp();
            else __syncthreads();
        }
    }
}

struct ReadQ8Args {
    uint64_t max_seq, start, n;  // positions [start, start + n) of every head
    const int32_t* lens;         // per sequence; NULL: all positions
    uint32_t heads, kv_heads, head_dim, nblk, shift;
};

// How many of the n positions of this sequence hold a token.
__device__ __forceinline__ uint64_t read_live(const ReadQ8Args& p, uint32_t bh) {
    if (!p.lens) return p.n;
    const int32_t l = p.lens[bh / p.kv_heads];
    if (l <= 0 || (uint64_t)l <= p.start) return 0;
    return (uint64_t)l - p.start < p.n ? (uint64_t)l - p.start : p.n;
}

// A CTA reads a run of one head's rows of k or of v, NC codes a thread: thread t
// keeps its place in the row (t mod head_dim / NC) and steps over the rows, so
// the places in memory take a few additions a vector; dividing a flat index for
// every vector instead took longer than HBM does (100 us for 8 sequences of
// 8192 x 8 heads x 128 against 51 us of bytes).  UNROLL rows are in flight.
template <typename T, int NC, int UNROLL>
__global__ void __launch_bounds__(256)
    kv_read_q8_vec_kernel(const int8_t* kc, const int8_t* vc, const float* ks, const float* vs, T* k, T* v,
                          ReadQ8Args p, uint32_t per_row, uint32_t rows, uint32_t runs) {
    pdl_begin();
    const uint32_t r0 = threadIdx.x / per_row, col = (threadIdx.x - r0 * per_row) * NC;
    if (r0 >= rows) return;  // threads beyond the last whole row of a step
    const uint32_t run = blockIdx.x % runs, hv = blockIdx.x / runs;  // run of rows; head of k or (behind them) v
    const bool is_v = hv >= p.heads;
    const uint32_t bh = is_v ? hv - p.heads : hv;
    const uint64_t live = read_live(p, bh);
    const int8_t* codes = (is_v ? vc : kc) + ((uint64_t)bh * p.max_seq + p.start) * p.head_dim + col;
    const float* scales = (is_v ? vs : ks) + (uint64_t)bh * p.nblk;
    T* out = (is_v ? v : k) + (uint64_t)bh * p.n * p.head_dim + col;
    const uint64_t at0 = (uint64_t)run * rows * UNROLL + r0;
    uint32_t c[UNROLL][NC / 4];
    float s[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const uint64_t at = at0 + (uint64_t)u * rows;
        s[u] = 0.0f;
#pragma unroll
        for (int e = 0; e < NC / 4; ++e) c[u][e] = 0;
        if (at < live) {
            q8_load(codes + at * p.head_dim, c[u]);
            s[u] = __ldg(scales + ((p.start + at) >> p.shift));
        }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const uint64_t at = at0 + (uint64_t)u * rows;
        if (at >= p.n) break;
        float x[NC];
#pragma unroll
        for (int e = 0; e < NC; e += 4) {
            float f[4];
            q8_unpack4(c[u][e / 4], f);
#pragma unroll
            for (int d = 0; d < 4; ++d) x[e + d] = fmul(f[d], s[u]);
        }
        q8_store_values(out + at * p.head_dim, x);
    }
}

template <typename T>
__global__ void __launch_bounds__(256)
    kv_read_q8_scalar_kernel(const int8_t* kc, const int8_t* vc, const float* ks, const float* vs, T* k, T* v,
                             ReadQ8Args p, uint64_t half) {
    pdl_begin();
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < 2 * half; i += (uint64_t)gridDim.x * 256) {
        const bool is_v = i >= half;
        const uint64_t r = is_v ? i - half : i, row = r / p.head_dim, bh = row / p.n, at = row - bh * p.n;
        float x = 0.0f;
        if (at < read_live(p, (uint32_t)bh)) {
            const uint64_t pos = p.start + at;
            x = fmul((float)(is_v ? vc : kc)[(bh * p.max_seq + pos) * p.head_dim + (r - row * p.head_dim)],
                     __ldg((is_v ? vs : ks) + bh * p.nblk + (pos >> p.shift)));
        }
        Vec<T>::store1((is_v ? v : k) + r, x);
    }
}

// log2 of a block size the caches can have, or -1.
int q8_block_shift(uint64_t block) {
    for (int s = 0; s <= 7; ++s)
        if (block == (1ull << s)) return s;
    return -1;
}

// Checks shared by the entry points of the int8 cache; OXIDE_OK or an error.
int q8_cache_check(const char* name, uint64_t batch, uint64_t kv_heads, uint64_t max_seq, uint64_t head_dim,
                   uint64_t block) {
    OXIDE_REQUIRE(q8_block_shift(block) >= 0, name, "block must be a power of two in [1, 128]");
    OXIDE_REQUIRE(head_dim < (1u << 16), name, "head_dim must be < 65536");
    OXIDE_REQUIRE(max_seq < (1ull << 31), name, "max_seq must be < 2^31");
    OXIDE_REQUIRE(batch < (1ull << 31) && kv_heads < (1ull << 31) && batch * kv_heads < (1ull << 31), name,
                  "batch * kv_heads must be < 2^31");
    // heads < 2^31, max_seq < 2^31: their product and the row bytes stay below 2^62 x 2^16
    OXIDE_REQUIRE(batch == 0 || kv_heads == 0 || head_dim == 0 ||
                      max_seq <= (UINT64_MAX >> 3) / head_dim / (batch * kv_heads), name, "cache size overflows");
    return OXIDE_OK;
}

static bool aligned_to(const void* p, uint64_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

template <typename T>
static int append_q8_entry(const char* name, int8_t* kc, int8_t* vc, float* ks, float* vs, const T* k, const T* v,
                           uint64_t batch, uint64_t kv_heads, uint64_t max_seq, uint64_t head_dim, uint64_t block,
                           uint64_t cur_len, const int32_t* cur_lens, uint64_t new_len, const int32_t* new_lens,
                           cudaStream_t st) {
    OXIDE_INJECT(name);
    if (int rc = q8_cache_check(name, batch, kv_heads, max_seq, head_dim, block)) return rc;
    OXIDE_REQUIRE(new_len <= max_seq && (cur_lens || cur_len <= max_seq - new_len), name,
                  "KV cache overflow: cur_len + new_len > max_seq");
    if (batch == 0 || kv_heads == 0 || new_len == 0 || head_dim == 0) return OXIDE_OK;
    OXIDE_REQUIRE(kc && vc && ks && vs && k && v, name, "null pointer");
    OXIDE_REQUIRE(kc != vc && ks != vs, name, "the key and value caches must not alias");
    constexpr uint64_t V = Vec<T>::N;
    AppendQ8Args p{};
    p.max_seq = (uint32_t)max_seq;
    p.cur_len = cur_lens ? 0u : (uint32_t)cur_len;
    p.new_len = (uint32_t)new_len;
    p.cur_lens = cur_lens;
    p.new_lens = new_lens;
    p.head_dim = (uint32_t)head_dim;
    p.shift = (uint32_t)q8_block_shift(block);
    p.nblk = (uint32_t)((max_seq + block - 1) / block);
    const uint64_t heads = batch * kv_heads;
    uint64_t wide = (new_len + block - 2) / block + 1;  // a run of new_len positions meets at most so many blocks
    if (wide > p.nblk) wide = p.nblk;
    const uint64_t items = 2 * heads * wide;
    OXIDE_REQUIRE(items < (1ull << 32), name, "too many blocks for one call (2^32): append fewer tokens at a time");
    p.half = (uint32_t)(heads * wide);
    p.items = (uint32_t)items;
    p.wide = FastDiv((uint32_t)wide);
    p.kv_heads = FastDiv((uint32_t)kv_heads);
    const uint64_t run = (block < new_len ? block : new_len) * head_dim;  // elements of the longest item
    const uint64_t cap = 1ull << 30, warps = (items + 7) / 8 < cap ? (items + 7) / 8 : cap,
                   ctas = items < cap ? items : cap;
    const bool vec = head_dim % V == 0 && aligned16(k) && aligned16(v) && aligned_to(kc, V) && aligned_to(vc, V) &&
                     run / V <= 4096;
    if (!vec) {
        if (run <= 1024) launch_k(kv_append_q8_scalar_kernel<T, 32>, (unsigned)warps, 256, 0, st, kc, vc, ks, vs, k, v, p);
        else launch_k(kv_append_q8_scalar_kernel<T, 256>, (unsigned)ctas, 256, 0, st, kc, vc, ks, vs, k, v, p);
    } else if (run / V <= 128) {
        launch_k(kv_append_q8_vec_kernel<T, 32, 4>, (unsigned)warps, 256, 0, st, kc, vc, ks, vs, k, v, p);
    } else if (run / V <= 1024) {
        launch_k(kv_append_q8_vec_kernel<T, 256, 4>, (unsigned)ctas, 256, 0, st, kc, vc, ks, vs, k, v, p);
    } else {
        launch_k(kv_append_q8_vec_kernel<T, 1024, 4>, (unsigned)ctas, 1024, 0, st, kc, vc, ks, vs, k, v, p);
    }
    return check_launch(name);
}

template <typename T>
static int read_q8_entry(const char* name, const int8_t* kc, const int8_t* vc, const float* ks, const float* vs, T* k,
                         T* v, uint64_t batch, uint64_t kv_heads, uint64_t max_seq, uint64_t head_dim, uint64_t block,
                         uint64_t start, uint64_t n, const int32_t* lens, cudaStream_t st) {
    OXIDE_INJECT(name);
    if (int rc = q8_cache_check(name, batch, kv_heads, max_seq, head_dim, block)) return rc;
    OXIDE_REQUIRE(n <= max_seq && start <= max_seq - n, name, "positions out of range: start + n > max_seq");
    if (batch == 0 || kv_heads == 0 || n == 0 || head_dim == 0) return OXIDE_OK;
    OXIDE_REQUIRE(kc && vc && ks && vs && k && v, name, "null pointer");
    OXIDE_REQUIRE(k != v, name, "the key and value outputs must not alias");
    constexpr uint64_t V = Vec<T>::N;
    ReadQ8Args p{};
    p.max_seq = max_seq;
    p.start = start;
    p.n = n;
    p.lens = lens;
    p.heads = (uint32_t)(batch * kv_heads);
    p.kv_heads = (uint32_t)kv_heads;
    p.head_dim = (uint32_t)head_dim;
    p.shift = (uint32_t)q8_block_shift(block);
    p.nblk = (uint32_t)((max_seq + block - 1) / block);
    const uint64_t cap = 1ull << 30;
    auto launch = [&](auto kern, uint64_t nc, uint64_t unroll) {
        const uint64_t per_row = head_dim / nc, rows = 256 / per_row;
        const uint64_t runs = (n + rows * unroll - 1) / (rows * unroll), ctas = 2ull * p.heads * runs;
        if (ctas >= (1ull << 31)) return false;
        launch_k(kern, (unsigned)ctas, 256, 0, st, kc, vc, ks, vs, k, v, p, (uint32_t)per_row, (uint32_t)rows, (uint32_t)runs);
        return true;
    };
    // Rows in flight a thread: 8 for long reads (ragged, 8192 x 64 heads x 128 bf16:
    // 62.8 us); 2 where eight would leave SMs without a CTA (1001 x 15 heads x 64 f32:
    // 3.9 us against 6.4).
    auto vec = [&](auto many, auto few, uint64_t nc) {
        const uint64_t steps = n * (head_dim / nc) / 256;  // per head
        return 2ull * p.heads * (steps / 8 + 1) >= 2ull * (uint64_t)sm_count() ? launch(many, nc, 8) : launch(few, nc, 2);
    };
    // 32 output bytes a thread, else 16 (odd multiples, other alignments).
    auto fits = [&](uint64_t nc) {
        return head_dim % nc == 0 && head_dim / nc <= 256 && aligned_to(k, nc * sizeof(T)) &&
               aligned_to(v, nc * sizeof(T)) && aligned_to(kc, nc) && aligned_to(vc, nc);
    };
    const bool done = (fits(2 * V) && vec(kv_read_q8_vec_kernel<T, 2 * V, 8>, kv_read_q8_vec_kernel<T, 2 * V, 2>, 2 * V)) ||
                      (fits(V) && vec(kv_read_q8_vec_kernel<T, V, 8>, kv_read_q8_vec_kernel<T, V, 2>, V));
    if (!done) {
        const uint64_t half = (uint64_t)p.heads * n * head_dim, want = (2 * half + 255) / 256;
        launch_k(kv_read_q8_scalar_kernel<T>, (unsigned)(want < cap ? want : cap), 256, 0, st, kc, vc, ks, vs, k, v, p, half);
    }
    return check_launch(name);
}

}  // namespace oxide

using oxide::bf16_t;

extern "C" {

int oxide_kv_cache_append_q8_f32(int8_t* k_cache, int8_t* v_cache, float* k_scale, float* v_scale, const float* k,
                                 const float* v, uint64_t batch, uint64_t kv_heads, uint64_t max_seq,
                                 uint64_t head_dim, uint64_t block, uint64_t cur_len, const int32_t* cur_lens,
                                 uint64_t new_len, const int32_t* new_lens, oxide_stream_t stream) {
    return oxide::append_q8_entry<float>("oxide_kv_cache_append_q8_f32", k_cache, v_cache, k_scale, v_scale, k, v,
                                         batch, kv_heads, max_seq, head_dim, block, cur_len, cur_lens, new_len,
                                         new_lens, stream);
}
int oxide_kv_cache_append_q8_bf16(int8_t* k_cache, int8_t* v_cache, float* k_scale, float* v_scale,
                                  const oxide_bf16* k, const oxide_bf16* v, uint64_t batch, uint64_t kv_heads,
                                  uint64_t max_seq, uint64_t head_dim, uint64_t block, uint64_t cur_len,
                                  const int32_t* cur_lens, uint64_t new_len, const int32_t* new_lens,
                                  oxide_stream_t stream) {
    return oxide::append_q8_entry<bf16_t>("oxide_kv_cache_append_q8_bf16", k_cache, v_cache, k_scale, v_scale, k, v,
                                          batch, kv_heads, max_seq, head_dim, block, cur_len, cur_lens, new_len,
                                          new_lens, stream);
}
int oxide_kv_cache_read_q8_f32(const int8_t* k_cache, const int8_t* v_cache, const float* k_scale,
                               const float* v_scale, float* k, float* v, uint64_t batch, uint64_t kv_heads,
                               uint64_t max_seq, uint64_t head_dim, uint64_t block, uint64_t start, uint64_t n,
                               const int32_t* lens, oxide_stream_t stream) {
    return oxide::read_q8_entry<float>("oxide_kv_cache_read_q8_f32", k_cache, v_cache, k_scale, v_scale, k, v, batch,
                                       kv_heads, max_seq, head_dim, block, start, n, lens, stream);
}
int oxide_kv_cache_read_q8_bf16(const int8_t* k_cache, const int8_t* v_cache, const float* k_scale,
                                const float* v_scale, oxide_bf16* k, oxide_bf16* v, uint64_t batch,
                                uint64_t kv_heads, uint64_t max_seq, uint64_t head_dim, uint64_t block,
                                uint64_t start, uint64_t n, const int32_t* lens, oxide_stream_t stream) {
    return oxide::read_q8_entry<bf16_t>("oxide_kv_cache_read_q8_bf16", k_cache, v_cache, k_scale, v_scale, k, v,
                                        batch, kv_heads, max_seq, head_dim, block, start, n, lens, stream);
}

}  // extern "C"
