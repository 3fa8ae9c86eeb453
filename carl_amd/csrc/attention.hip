// attention.hip - linear attention with a decay for each head: the C-ABI's
// checks and passes, the joining of split sequences, the sums over query heads
// that share a key head, and the recurrent form.  The chunked kernel is in
// attention_kernel.h, its mathematics in attention.h.
#include <algorithm>
#include <cstring>

#include "attention.h"
#include "status.h"

using namespace carl;

int carl::launchAttention(int type, const Pass& pass, int firstRole, int roles, bool states, hipStream_t stream)
{
    if (type == CARL_OP_F32) return launchAttentionOf<float>(pass, firstRole, roles, states, stream);
    if (type == CARL_OP_BF16) return launchAttentionOf<bf16>(pass, firstRole, roles, states, stream);
    return launchAttentionOf<f16>(pass, firstRole, roles, states, stream);
}

namespace {

// The memories before each segment from what each leaves, in the place of the
// latter.  A thread for each element of a memory; eight segments' loads are on
// their way at once, since each one's store would hold back the next one's
// (36 segments of 64 x 128, 16 units: 25 us one by one).
__global__ __launch_bounds__(256) void joinKernel(const Pass pass)
{
    constexpr int kAtOnce = 8;
    const Role& r = pass.role[blockIdx.z];
    const int64_t size = (int64_t)r.dimA * r.dimC, units = pass.batch * pass.heads;
    const int64_t unit = blockIdx.x;
    for (int64_t e = threadIdx.x + (int64_t)blockIdx.y * 256; e < size; e += (int64_t)gridDim.y * 256) {
        const int64_t swapped = e % r.dimC * r.dimA + e / r.dimC;
        float m = r.first ? r.first[unit * size + (r.firstSwapped ? swapped : e)] : 0.0f;
        for (int i0 = 0; i0 < pass.segments; i0 += kAtOnce) {
            float own[kAtOnce], f[kAtOnce];
#pragma unroll
            for (int j = 0; j < kAtOnce; j++) {
                const int i = i0 + j < pass.segments ? i0 + j : pass.segments - 1;
                const int64_t at = (r.backwards ? pass.segments - 1 - i : i) * units + unit;
                own[j] = r.parts[at * size + e];
                f[j] = r.factors[at];
            }
#pragma unroll
            for (int j = 0; j < kAtOnce; j++) {
                const int i = i0 + j;
                if (i >= pass.segments) break;
                r.parts[((r.backwards ? pass.segments - 1 - i : i) * units + unit) * size + e] = m;
                m = signbit(f[j]) ? own[j] : m * f[j] + own[j];       // nothing of a memory that an episode's start clears
            }
        }
        if (r.last) r.last[unit * size + (r.lastSwapped ? swapped : e)] = m;
    }
}

// Sums of `group` query heads' float32 rows into their shared head's row, of
// the keys' and of the values' gradients.  A workgroup for each step of a
// sequence; four elements a thread where all rows allow it.
struct GroupSum {
    const float* rows;          // [batch, steps, heads * group, dim]
    Rows out;
    int32_t dim, wide;
};
struct GroupSums {
    GroupSum sum[2];
    int64_t steps;
    int32_t heads, group;
};

template <typename T> __global__ __launch_bounds__(256) void groupKernel(const GroupSums args)
{
    const GroupSum& s = args.sum[blockIdx.z];
    const int64_t batch = blockIdx.y;
    const int width = s.wide ? 4 : 1, each = s.dim / width;
    for (int64_t step = blockIdx.x; step < args.steps; step += gridDim.x) {
        const float* rows = s.rows + (batch * args.steps + step) * args.heads * args.group * s.dim;
        T* out = static_cast<T*>(s.out.data) + batch * s.out.batch + step * s.out.step;
        for (int e = threadIdx.x; e < args.heads * each; e += 256) {
            const int head = e / each, d = (e - head * each) * width;
            const float* from = rows + (int64_t)head * args.group * s.dim + d;
            T* to = out + head * s.out.head + d;
            if (s.wide) {
                f32x4 sum = *reinterpret_cast<const f32x4*>(from);
                for (int g = 1; g < args.group; g++) sum += *reinterpret_cast<const f32x4*>(from + g * s.dim);
                *reinterpret_cast<vec<T, 4>*>(to) = fromFloat<T, 4>(sum);
            } else {
                float sum = *from;
                for (int g = 1; g < args.group; g++) sum += from[g * s.dim];
                *to = (T)sum;
            }
        }
    }
}

// ---- the recurrent form ------------------------------------------------------
// Bound by the memory's bytes, read and written once: each wave takes a tile of
// 32 columns (8 lanes of 16 bytes) of one head's memory and its rows 8 at a
// time, so a wave's accesses are whole 128-byte lines and nothing has to be
// exchanged but the 8 partial sums of an output.  131,072 agents, 4 heads of 32
// in float32: 816 us, 5.6 TB/s; 34 agents: 5.9 us, a launch's latency.
struct Step {
    Rows q, k, v, out;
    const float* logDecay;
    const uint8_t* starts;
    int64_t startsBatch;
    float* state;
    int64_t batch;
    int32_t heads, group, dimK, dimV;
    int32_t wide;
    float scale;
};

template <typename T> __global__ __launch_bounds__(256) void stepKernel(const Step p, const int64_t waves, const int tiles)
{
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (w >= waves) return;
    const int tile = (int)(w % tiles), head = (int)(w / tiles % p.heads);
    const int64_t batch = w / tiles / p.heads;
    const int lane = threadIdx.x & 63, y = tile * 32 + (lane & 7) * 4, first = lane >> 3;
    const int have = y >= p.dimV ? 0 : p.dimV - y < 4 ? p.dimV - y : 4;
    const bool fresh = p.starts && p.starts[batch * p.startsBatch] != 0;
    const float decay = expf(p.logDecay[head]);
    const T* q = static_cast<const T*>(p.q.data) + batch * p.q.batch + head * p.q.head;
    const T* k = static_cast<const T*>(p.k.data) + batch * p.k.batch + head / p.group * p.k.head;
    const T* v = static_cast<const T*>(p.v.data) + batch * p.v.batch + head / p.group * p.v.head;
    float* state = p.state + (batch * p.heads + head) * (int64_t)p.dimK * p.dimV;
    f32x4 value = { 0.f, 0.f, 0.f, 0.f }, out = { 0.f, 0.f, 0.f, 0.f };
    for (int i = 0; i < 4; i++)
        if (i < have) value[i] = (float)v[y + i];
    for (int x0 = 0; x0 < p.dimK; x0 += 32) {
        f32x4 m[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int x = x0 + u * 8 + first;
            m[u] = f32x4{ 0.f, 0.f, 0.f, 0.f };
            if (fresh || x >= p.dimK) continue;
            const float* s = state + (int64_t)x * p.dimV + y;
            if (p.wide && have == 4) m[u] = *reinterpret_cast<const f32x4*>(s);
            else
                for (int i = 0; i < 4; i++)
                    if (i < have) m[u][i] = s[i];
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int x = x0 + u * 8 + first;
            if (x >= p.dimK) continue;
            const float key = (float)k[x], query = (float)q[x];
            m[u] = fresh ? value * key : m[u] * decay + value * key;
            out += m[u] * query;
            float* s = state + (int64_t)x * p.dimV + y;
            if (p.wide && have == 4) *reinterpret_cast<f32x4*>(s) = m[u];
            else
                for (int i = 0; i < 4; i++)
                    if (i < have) s[i] = m[u][i];
        }
    }
    for (int i = 0; i < 4; i++)
        for (int d = 8; d < 64; d <<= 1) out[i] += __shfl_xor(out[i], d);
    if (first != 0) return;
    T* to = static_cast<T*>(p.out.data) + batch * p.out.batch + head * p.out.head + y;
    for (int i = 0; i < 4; i++)
        if (i < have) to[i] = (T)(out[i] * p.scale);
}

// ---- checks ------------------------------------------------------------------

constexpr int64_t kMostUnits = (int64_t)1 << 22;     // three workgroups each: 3 x 2^30 threads a launch

int elementBytes(int type) { return type == CARL_OP_F32 ? 4 : 2; }

bool empty(const carl_attention& a) { return a.batch == 0 || a.steps == 0; }

int checkAttention(const carl_attention* a, bool backward, bool step)
{
    if (!a) return fail(CARL_ERR_VALUE, "null attention argument");
    if (a->type != CARL_OP_F32 && a->type != CARL_OP_BF16 && a->type != CARL_OP_F16) return fail(CARL_ERR_TYPE, "unknown element type");
    if (a->batch < 0 || a->steps < 0) return fail(CARL_ERR_VALUE, "batch and steps must be non-negative");
    if (step && a->steps != 1) return fail(CARL_ERR_VALUE, "steps must be 1");
    if (a->heads < 1 || a->heads > 65535) return fail(CARL_ERR_VALUE, "heads must be in [1, 65535]");
    if (a->kv_heads < 1 || a->heads % a->kv_heads) return fail(CARL_ERR_VALUE, "heads must be a multiple of kv_heads");
    if (a->key_dim < 1 || a->key_dim > CARL_ATTENTION_MAX_DIM) return fail(CARL_ERR_VALUE, "key_dim must be in [1, 128]");
    if (a->value_dim < 1 || a->value_dim > CARL_ATTENTION_MAX_DIM) return fail(CARL_ERR_VALUE, "value_dim must be in [1, 128]");
    if (a->batch > kMostUnits / a->heads) return fail(CARL_ERR_VALUE, "batch times heads must be at most 4,194,304");
    if (a->steps > (int64_t)1 << 40) return fail(CARL_ERR_VALUE, "too many steps");
    if (a->batch > 0 && !a->log_decay) return fail(CARL_ERR_VALUE, "null log_decay");
    if (empty(*a)) return CARL_OK;
    if (!a->q.data || !a->k.data || !a->v.data) return fail(CARL_ERR_VALUE, "null attention input");
    if (!backward && !a->out.data) return fail(CARL_ERR_VALUE, "null attention output");
    if (backward && (!a->d_out.data || !a->d_q.data || !a->d_k.data || !a->d_v.data))
        return fail(CARL_ERR_VALUE, "null attention gradient");
    return CARL_OK;
}

// ---- passes ------------------------------------------------------------------

// Bytes that every row's address is a multiple of (at most 16): the row
// strides that are taken more than once and the base.
int grainOf(const Rows& r, int type, int64_t batch, int64_t steps, int heads)
{
    const int size = elementBytes(type);
    uint64_t bits = reinterpret_cast<uintptr_t>(r.data) | 16;
    if (batch > 1) bits |= (uint64_t)r.batch * size;
    if (steps > 1) bits |= (uint64_t)r.step * size;
    if (heads > 1) bits |= (uint64_t)r.head * size;
    return (int)(bits & (~bits + 1));
}

// The same for rows of `dim` elements that are read; 0 where 64 of them do not
// lie within 32 bits.
int readGrain(const Rows& r, int type, int64_t batch, int64_t steps, int heads, int dim)
{
    const int size = elementBytes(type);
    if (r.step < 0 || 63 * r.step * size + dim * size > 0xffffff00ll) return 0;
    const int grain = grainOf(r, type, batch, steps, heads), width = dim * size & -(dim * size);
    return grain < width ? grain : width;
}

Rows rowsOf(const carl_rows& r) { return Rows{ r.data, r.batch, r.step, r.head }; }

// How a sequence is split.  One workgroup walks a whole sequence of one head
// where those and the pass's directions fill the GPU; with fewer, segments of
// about 256 steps or more (never under 192, in whole 64s), as many as run at once
// (two workgroups a compute unit with the widest rows, three or four with
// others).  Backwards that counts all three directions, as they run where the
// widths of keys and values are equal; where they differ run() launches them
// one after the other, and each has fewer workgroups than would fit.  Segments
// need the memories before them, which a first launch sums up (reading keys and
// values once more) and a second joins.  6 sequences of 4,603 steps, 8 heads of
// 128: 18 segments both ways, as 1,024 workgroups would have them, 855 us with
// gradients; as here 617.
//
// Backwards fewer directions are summed up than run, and the first launch would
// leave compute units with one workgroup: it takes the segments in two halves
// where all of them run at once (three workgroups a compute unit, or as many
// as of the others) and their length allows it, a multiple of 128: 6 x 4,603
// (segments of 1,536) with gradients 636 us with whole segments, 601 with
// halves, when that was measured.
struct Split {
    int segments;
    int64_t steps;
    int finer;
};

Split splitOf(const carl_attention& a, bool backward)
{
    const int64_t units = a.batch * a.heads * (backward ? 3 : 1);
    const int widest = std::max(a.key_dim, a.value_dim), other = std::min(a.key_dim, a.value_dim);
    const int64_t resident = 256 * (other > 64 ? 2 : widest > 64 ? 3 : a.type == CARL_OP_F32 ? 2 : 4);
    if (units > resident / 2 || a.steps <= 256) return { 1, std::max<int64_t>(a.steps, 1), 1 };
    int64_t segments = std::min<int64_t>(resident / units, (a.steps + 255) / 256);
    int64_t steps = (a.steps + segments - 1) / segments;
    steps = (steps + 63) / 64 * 64;
    segments = (a.steps + steps - 1) / steps;
    const int64_t summed = a.batch * a.heads * (backward ? 2 : 1) * segments;
    const bool halves = steps % 128 == 0 && steps >= 512 && summed * 2 <= std::max<int64_t>(resident, 256 * 3);
    return { (int)segments, steps, halves ? 2 : 1 };
}

int64_t rounded(int64_t bytes) { return (bytes + 255) / 256 * 256; }

struct Layout {
    int64_t parts = 0, factors = 0;      // bytes of one role's
    int64_t keyRows = 0, valueRows = 0;  // of the query heads' gradients
    int64_t total = 0;
};

Layout layoutOf(const carl_attention& a, bool backward)
{
    Layout l;
    const Split s = splitOf(a, backward);
    if (s.segments > 1) {
        const int64_t units = a.batch * a.heads * s.segments * s.finer;
        l.parts = rounded(units * a.key_dim * a.value_dim * 4);
        l.factors = rounded(units * 4);
    }
    if (backward && a.heads != a.kv_heads) {
        l.keyRows = rounded(a.batch * a.steps * a.heads * a.key_dim * 4);
        l.valueRows = rounded(a.batch * a.steps * a.heads * a.value_dim * 4);
    }
    l.total = (l.parts + l.factors) * (backward ? 2 : 1) + l.keyRows + l.valueRows;
    return l;
}

void dealUnits(Pass& pass)
{
    // (the grid's second dimension holds 65,535)
    const int64_t groups = pass.batch * pass.segments;
    pass.dealGroups = groups >= 64 && groups <= 8 * 65535;
}

// `summed`: the first roles, which have parts of their own.
int run(const carl_attention& a, Pass& pass, int summed, int roles, hipStream_t stream)
{
    // roles next to each other with the same widths share a launch
    const auto launch = [&](const Pass& pass, bool states, int roles) {
        for (int i = 0; i < roles;) {
            int n = 1;
            while (i + n < roles && pass.role[i + n].dimA == pass.role[i].dimA && pass.role[i + n].dimC == pass.role[i].dimC) n++;
            if (int rc = launchAttention(a.type, pass, i, n, states, stream)) return rc;
            i += n;
        }
        return (int)CARL_OK;
    };
    if (pass.segments > 1) {
        Pass sums = pass;       // an empty last half leaves a memory of zeros and a factor of one
        sums.segments *= pass.finer;
        sums.segmentSteps /= pass.finer;
        dealUnits(sums);
        if (int rc = launch(sums, true, summed)) return rc;
        const int blocks = (int)(((int64_t)a.key_dim * a.value_dim + 255) / 256);
        joinKernel<<<dim3((unsigned)(a.batch * a.heads), (unsigned)blocks, (unsigned)summed), 256, 0, stream>>>(sums);
        if (int rc = launched("joining of segments")) return rc;
    }
    return launch(pass, false, roles);
}

Pass passOf(const carl_attention& a, bool backward)
{
    Pass pass{};
    const Split s = splitOf(a, backward);
    pass.batch = a.batch;
    pass.steps = a.steps;
    pass.heads = a.heads;
    pass.segments = s.segments;
    pass.segmentSteps = s.steps;
    pass.finer = s.finer;
    dealUnits(pass);
    pass.logDecay = a.log_decay;
    pass.starts = a.starts;
    pass.startsBatch = a.starts_batch;
    pass.startsStep = a.starts_step;
    return pass;
}

// which: 0 query-like rows [heads], 1 key or value rows [kv_heads]
Role roleOf(const carl_attention& a, const carl_rows& x, bool xShared, const carl_rows& y, bool yShared, const carl_rows& z,
            bool zShared, const Rows& out, int dimA, int dimC)
{
    Role r{};
    const int group = a.heads / a.kv_heads;
    r.a = rowsOf(x);
    r.b = rowsOf(y);
    r.c = rowsOf(z);
    r.out = out;
    r.aHeads = xShared ? group : 1;
    r.bHeads = yShared ? group : 1;
    r.cHeads = zShared ? group : 1;
    r.aGrain = readGrain(r.a, a.type, a.batch, a.steps, xShared ? a.kv_heads : a.heads, dimA);
    r.bGrain = readGrain(r.b, a.type, a.batch, a.steps, yShared ? a.kv_heads : a.heads, dimA);
    r.cGrain = readGrain(r.c, a.type, a.batch, a.steps, zShared ? a.kv_heads : a.heads, dimC);
    r.outWide = dimC % 4 == 0 && grainOf(out, a.type, a.batch, a.steps, a.heads) >= 4 * elementBytes(a.type);
    r.dimA = dimA;
    r.dimC = dimC;
    r.scaleP = a.scale;
    r.inShift = 1;
    return r;
}


__global__ __launch_bounds__(256) void copyKernel(const float* from, float* to, int64_t n)
{
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n; e += (int64_t)gridDim.x * 256)
        to[e] = from ? from[e] : 0.0f;
}

// a sequence of no steps leaves the memory as it was
int passMemory(const float* from, float* to, int64_t n, hipStream_t stream)
{
    if (!to || n == 0) return CARL_OK;
    copyKernel<<<dim3((unsigned)std::min<int64_t>((n + 255) / 256, 4096)), 256, 0, stream>>>(from, to, n);
    return launched("memory copy");
}

}  // namespace

extern "C" {

int carl_linear_attention_workspace(const carl_attention* a, int backward, int64_t* bytes)
{
    if (!a || !bytes) return fail(CARL_ERR_VALUE, "null attention argument");
    carl_attention shape = *a;
    // sizes only: pointers may not be there yet
    static char some;
    static const float none = 0.0f;
    shape.log_decay = &none;
    for (carl_rows* r : { &shape.q, &shape.k, &shape.v, &shape.out, &shape.d_out, &shape.d_q, &shape.d_k, &shape.d_v }) r->data = &some;
    if (int rc = checkAttention(&shape, backward != 0, false)) return rc;
    *bytes = empty(shape) ? 0 : layoutOf(shape, backward != 0).total;
    return CARL_OK;
}

int carl_linear_attention(const carl_attention* a, void* stream)
{
    if (int rc = checkAttention(a, false, false)) return rc;
    const int64_t memory = a->batch * a->heads * a->key_dim * a->value_dim;
    if (empty(*a)) return passMemory(a->initial_state, a->final_state, memory, (hipStream_t)stream);
    const Layout l = layoutOf(*a, false);
    if (l.total > 0 && !a->workspace) return fail(CARL_ERR_VALUE, "null workspace");
    Pass pass = passOf(*a, false);
    Role& r = pass.role[0];
    r = roleOf(*a, a->q, false, a->k, true, a->v, true, rowsOf(a->out), a->key_dim, a->value_dim);
    r.scaleIn = a->scale;
    r.scaleOut = 1.0f;
    r.first = a->initial_state;
    r.last = a->final_state;
    r.parts = static_cast<float*>(a->workspace);
    r.factors = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + l.parts);
    return run(*a, pass, 1, 1, (hipStream_t)stream);
}

int carl_linear_attention_backward(const carl_attention* a, void* stream)
{
    if (int rc = checkAttention(a, true, false)) return rc;
    const int64_t memory = a->batch * a->heads * a->key_dim * a->value_dim;
    if (empty(*a)) return passMemory(a->d_final_state, a->d_initial_state, memory, (hipStream_t)stream);
    const Layout l = layoutOf(*a, true);
    if (l.total > 0 && !a->workspace) return fail(CARL_ERR_VALUE, "null workspace");
    Pass pass = passOf(*a, true);
    char* work = static_cast<char*>(a->workspace);
    const bool grouped = a->heads != a->kv_heads;
    const auto queryRows = [&](int64_t at, int dim) {
        return Rows{ work + at, a->steps * a->heads * dim, (int64_t)a->heads * dim, dim };
    };
    const int64_t rowsAt = (l.parts + l.factors) * 2;
    const Rows keyRows = grouped ? queryRows(rowsAt, a->key_dim) : rowsOf(a->d_k);
    const Rows valueRows = grouped ? queryRows(rowsAt + l.keyRows, a->value_dim) : rowsOf(a->d_v);

    // dq: time forwards, the memory transposed
    Role& dq = pass.role[0];
    dq = roleOf(*a, a->d_out, false, a->v, true, a->k, true, rowsOf(a->d_q), a->value_dim, a->key_dim);
    dq.scaleIn = a->scale;
    dq.scaleOut = 1.0f;
    dq.first = a->initial_state;
    dq.firstSwapped = 1;
    // dk and dv: time backwards, the gradient of the memory instead of it
    Role& dk = pass.role[2];
    dk = roleOf(*a, a->v, true, a->d_out, false, a->q, false, keyRows, a->value_dim, a->key_dim);
    Role& dv = pass.role[1];
    dv = roleOf(*a, a->k, true, a->q, false, a->d_out, false, valueRows, a->key_dim, a->value_dim);
    for (Role* r : { &dk, &dv }) {
        r->backwards = 1;
        r->inShift = 0;
        r->scaleIn = 1.0f;
        r->scaleOut = a->scale;
        r->first = a->d_final_state;
        r->outFloat = grouped;
    }
    dk.firstSwapped = 1;
    dv.last = a->d_initial_state;
    for (int i = 0; i < 2; i++) {
        pass.role[i].parts = reinterpret_cast<float*>(work + (l.parts + l.factors) * i);
        pass.role[i].factors = reinterpret_cast<float*>(work + (l.parts + l.factors) * i + l.parts);
    }
    dk.parts = dv.parts;        // dk's memory is dv's, transposed
    dk.partsSwapped = 1;
    if (int rc = run(*a, pass, 2, 3, (hipStream_t)stream)) return rc;
    if (!grouped) return CARL_OK;
    GroupSums sums{};
    sums.steps = a->steps;
    sums.heads = a->kv_heads;
    sums.group = a->heads / a->kv_heads;
    const auto sumOf = [&](const Rows& from, const carl_rows& to, int dim) {
        const Rows out = rowsOf(to);
        const bool wide = dim % 4 == 0 && grainOf(out, a->type, a->batch, a->steps, a->kv_heads) >= 4 * elementBytes(a->type);
        return GroupSum{ static_cast<const float*>(from.data), out, dim, wide };
    };
    sums.sum[0] = sumOf(keyRows, a->d_k, a->key_dim);
    sums.sum[1] = sumOf(valueRows, a->d_v, a->value_dim);
    // (65,535 sequences at a time: the grid's second dimension)
    for (int64_t first = 0; first < a->batch; first += 65535) {
        GroupSums some = sums;
        for (GroupSum& s : some.sum) {
            s.rows += first * a->steps * a->heads * s.dim;
            s.out.data = static_cast<char*>(s.out.data) + first * s.out.batch * elementBytes(a->type);
        }
        const dim3 grid((unsigned)std::min<int64_t>(a->steps, 1 << 20), (unsigned)std::min<int64_t>(a->batch - first, 65535), 2);
        const hipStream_t s = (hipStream_t)stream;
        if (a->type == CARL_OP_F32) groupKernel<float><<<grid, 256, 0, s>>>(some);
        else if (a->type == CARL_OP_BF16) groupKernel<bf16><<<grid, 256, 0, s>>>(some);
        else groupKernel<f16><<<grid, 256, 0, s>>>(some);
        if (int rc = launched("sum over shared heads")) return rc;
    }
    return CARL_OK;
}

int carl_linear_attention_step(const carl_attention* a, float* state, void* stream)
{
    if (int rc = checkAttention(a, false, true)) return rc;
    if (a->batch == 0) return CARL_OK;
    if (!state) return fail(CARL_ERR_VALUE, "null state");
    const int tiles = (a->value_dim + 31) / 32;
    const int64_t waves = a->batch * a->heads * tiles;
    Step p{};
    p.q = rowsOf(a->q);
    p.k = rowsOf(a->k);
    p.v = rowsOf(a->v);
    p.out = rowsOf(a->out);
    p.logDecay = a->log_decay;
    p.starts = a->starts;
    p.startsBatch = a->starts_batch;
    p.state = state;
    p.batch = a->batch;
    p.heads = a->heads;
    p.group = a->heads / a->kv_heads;
    p.dimK = a->key_dim;
    p.dimV = a->value_dim;
    p.wide = a->value_dim % 4 == 0 && reinterpret_cast<uintptr_t>(state) % 16 == 0;
    p.scale = a->scale;
    const dim3 grid((unsigned)((waves + 3) / 4));
    const hipStream_t s = (hipStream_t)stream;
    if (a->type == CARL_OP_F32) stepKernel<float><<<grid, 256, 0, s>>>(p, waves, tiles);
    else if (a->type == CARL_OP_BF16) stepKernel<bf16><<<grid, 256, 0, s>>>(p, waves, tiles);
    else stepKernel<f16><<<grid, 256, 0, s>>>(p, waves, tiles);
    return launched("linear attention step");
}

}  // extern "C"
