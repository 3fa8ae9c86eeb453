// ffn.hip - the gated feed-forward block: the C-ABI's checks, operands that
// have to be laid out, and the passes of ffn.h.
#include <algorithm>

#include "ffn.h"
#include "status.h"

using namespace carl;

int carl::outerTile(int m, int n) { return m > 128 && n > 128 ? 256 : 128; }

namespace {

int elementBytes(int type) { return type == CARL_OP_F32 ? 4 : 2; }
int64_t upTo(int64_t x, int64_t multiple) { return (x + multiple - 1) / multiple * multiple; }

constexpr int64_t kMostRows = (int64_t)1 << 28;

// Of a product's launch, at most, where it is a large one: launchProduct()
// then takes tiles of at least 128 x 64 (float32, 256 threads) or 128 x 128
// (16 bits, 512 threads), a multiple of 8 of them across the rows.
int64_t threadsOf(const carl_ffn& f)
{
    const bool wide = f.type == CARL_OP_F32;
    const int64_t columns = std::max(f.width, f.inner), tile = wide ? 64 : 128;
    return upTo((f.rows + 127) / 128, 8) * ((columns + tile - 1) / tile) * (wide ? 256 : 512);
}

int checkFfn(const carl_ffn* f, bool backward)
{
    if (!f) return fail(CARL_ERR_VALUE, "null feed-forward argument");
    if (f->type != CARL_OP_F32 && f->type != CARL_OP_BF16 && f->type != CARL_OP_F16) return fail(CARL_ERR_TYPE, "unknown element type");
    if (f->activation != CARL_SILU && f->activation != CARL_GELU) return fail(CARL_ERR_VALUE, "unknown activation");
    if (f->width < 1 || f->width > CARL_FFN_MAX_DIM) return fail(CARL_ERR_VALUE, "width must be in [1, 65536]");
    if (f->inner < 1 || f->inner > CARL_FFN_MAX_DIM) return fail(CARL_ERR_VALUE, "inner must be in [1, 65536]");
    if (f->rows < 0 || f->rows > kMostRows || threadsOf(*f) > (int64_t)1 << 31) return fail(CARL_ERR_VALUE, "rows are out of range");
    if (!f->w_gate || !f->w_up || !f->w_down) return fail(CARL_ERR_VALUE, "null weights");
    if (f->rows == 0) return CARL_OK;
    if (!f->x || (!backward && !f->y) || (backward && !f->dy)) return fail(CARL_ERR_VALUE, "null feed-forward tensor");
    return CARL_OK;
}

// Where a pass's operands lie: in place where the copies into LDS can take
// them (16-byte pieces of aligned rows), else in the workspace, padded.
class Plan {
public:
    Plan(int type, char* workspace) : size_(elementBytes(type)), piece_(16 / size_), work_(workspace) {}

    int64_t bytes() const { return at_; }
    const PackArgs& packs() const { return packs_; }

    void* take(int64_t bytes)
    {
        void* p = work_ ? work_ + at_ : nullptr;
        at_ += upTo(bytes, 256);
        return p;
    }

    Panel rows(const void* data, int64_t rows, int64_t cols, int64_t stride)
    {
        const bool fits = reinterpret_cast<uintptr_t>(data) % 16 == 0 && stride % piece_ == 0 && cols % piece_ == 0
                       && stride >= cols && stride <= ((int64_t)1 << 22) / size_;
        if (fits) return Panel{ data, rows, stride, (int32_t)cols };
        const int64_t to = upTo(cols, piece_);
        return pack({ data, take(rows * to * size_), rows, cols, stride, to, 0 }, rows);
    }

    // the transpose of a [rows, cols] matrix
    Panel transposed(const void* data, int64_t rows, int64_t cols)
    {
        const int64_t to = upTo(rows, piece_);
        return pack({ data, take(cols * to * size_), rows, cols, cols, to, 1 }, cols);
    }

    Panel scratch(int64_t rows, int64_t cols)
    {
        const int64_t stride = upTo(cols, 64);
        return Panel{ take(rows * stride * size_), rows, stride, (int32_t)upTo(cols, piece_) };
    }

private:
    Panel pack(const PackJob& job, int64_t rows)
    {
        packs_.job[packs_.jobs++] = job;
        return Panel{ job.to, rows, job.toStride, (int32_t)job.toStride };
    }

    int64_t size_, piece_;
    char* work_;
    int64_t at_ = 0;
    PackArgs packs_{};
};

// float16: where the factors of h, dg and du are.
ScaleArgs scalesOf(const carl_ffn& f, Plan& plan)
{
    ScaleArgs a{};
    if (f.type != CARL_OP_F16) return a;
    a.part = static_cast<float*>(plan.take(5 * kScaleBlocks * 4));
    a.scale = static_cast<float*>(plan.take(4 * 4));
    return a;
}

const float* factor(const ScaleArgs& a, int which) { return a.scale ? a.scale + which : nullptr; }

// Up to so many rows the forward pass is a matter of latency.
constexpr int kThinRows = 128;

struct Forward {
    Panel x{}, gate{}, up{}, down{}, h;
    ScaleArgs scales{};
    explicit Forward(const carl_ffn& f, Plan& plan)
    {
        if (f.rows <= kThinRows) {
            const int64_t stride = upTo(f.inner, 64);
            h = Panel{ plan.take(f.rows * stride * 4), f.rows, stride, f.inner };
            return;
        }
        x = plan.rows(f.x, f.rows, f.width, f.x_row);
        gate = plan.rows(f.w_gate, f.inner, f.width, f.width);
        up = plan.rows(f.w_up, f.inner, f.width, f.width);
        down = plan.rows(f.w_down, f.width, f.inner, f.inner);
        h = plan.scratch(f.rows, f.inner);
        scales = scalesOf(f, plan);
        scales.panels = 3;
        scales.rows[0] = x;
        scales.rows[1] = gate;
        scales.rows[2] = up;
    }
};

struct Backward {
    Panel x, dy, gate, up, downT, gateT{}, upT{}, h, dg, du;
    ScaleArgs scales{};
    OuterArgs outer{};
    int tile = 256;
    explicit Backward(const carl_ffn& f, Plan& plan)
    {
        x = plan.rows(f.x, f.rows, f.width, f.x_row);
        dy = plan.rows(f.dy, f.rows, f.width, f.dy_row);
        gate = plan.rows(f.w_gate, f.inner, f.width, f.width);
        up = plan.rows(f.w_up, f.inner, f.width, f.width);
        downT = plan.transposed(f.w_down, f.width, f.inner);
        gateT = plan.transposed(f.w_gate, f.inner, f.width);
        upT = plan.transposed(f.w_up, f.inner, f.width);
        h = plan.scratch(f.rows, f.inner);
        dg = plan.scratch(f.rows, f.inner);
        du = plan.scratch(f.rows, f.inner);
        scales = scalesOf(f, plan);
        scales.panels = 5;
        const Panel normed[5] = { x, gate, up, dy, downT };
        std::copy(normed, normed + 5, scales.rows);

        // the three weights' gradients in one launch, rows split until the
        // tiles fill the compute units
        outer.k = f.rows;
        outer.jobs = 3;
        tile = outerTile(f.width, f.inner);
        const Panel p[3] = { dg, du, dy }, q[3] = { x, x, h };
        int tiles = 0;
        for (int j = 0; j < 3; j++) {
            outer.p[j] = p[j];
            outer.q[j] = q[j];
            outer.m[j] = j < 2 ? f.inner : f.width;
            outer.n[j] = j < 2 ? f.width : f.inner;
            tiles += ((outer.m[j] + tile - 1) / tile) * ((outer.n[j] + tile - 1) / tile);
        }
        const int64_t step = 128 / elementBytes(f.type);
        const int64_t splits = std::max<int64_t>(1, std::min<int64_t>((tile == 256 ? 256 : 512) / tiles, f.rows / (8 * step)));
        outer.splitRows = upTo((f.rows + splits - 1) / splits, step);
        outer.splits = (int)((f.rows + outer.splitRows - 1) / std::max<int64_t>(outer.splitRows, 1));
        for (int j = 0; j < 3; j++)
            outer.part[j] = static_cast<float*>(plan.take((int64_t)outer.splits * f.width * f.inner * 4));
    }
};

int product(int type, int kind, const ProductArgs& a, hipStream_t s)
{
    if (type == CARL_OP_F32) return launchProduct<float>(kind, a, s);
    if (type == CARL_OP_BF16) return launchProduct<bf16>(kind, a, s);
    return launchProduct<f16>(kind, a, s);
}

int thin(int type, bool gate, const ThinArgs& a, hipStream_t s)
{
    if (type == CARL_OP_F32) return launchThin<float>(gate, a, s);
    if (type == CARL_OP_BF16) return launchThin<bf16>(gate, a, s);
    return launchThin<f16>(gate, a, s);
}

int pack(int type, const PackArgs& a, hipStream_t s)
{
    if (a.jobs == 0) return CARL_OK;
    if (type == CARL_OP_F32) return launchPack<float>(a, s);
    if (type == CARL_OP_BF16) return launchPack<bf16>(a, s);
    return launchPack<f16>(a, s);
}

int outerProducts(int type, const OuterArgs& a, int tile, hipStream_t s)
{
    if (type == CARL_OP_F32) return launchOuter<float>(a, tile, s);
    if (type == CARL_OP_BF16) return launchOuter<bf16>(a, tile, s);
    return launchOuter<f16>(a, tile, s);
}

int scale(int type, const ScaleArgs& a, hipStream_t s) { return type == CARL_OP_F16 ? launchScale(a, s) : (int)CARL_OK; }

int sums(int type, const SumArgs& a, hipStream_t s)
{
    if (type == CARL_OP_F32) return launchSum<float>(a, s);
    if (type == CARL_OP_BF16) return launchSum<bf16>(a, s);
    return launchSum<f16>(a, s);
}

// A plain product into the caller's [rows, width] matrix.
ProductArgs toRows(const carl_ffn& f, void* out)
{
    ProductArgs a{};
    a.m = f.rows;
    a.n = f.width;
    a.out[0] = out;
    a.outStride = a.outWidth = f.width;
    a.outWide = reinterpret_cast<uintptr_t>(out) % 16 == 0 && f.width * elementBytes(f.type) % 16 == 0;
    return a;
}

}  // namespace

extern "C" {

int carl_gated_ffn_workspace(const carl_ffn* f, int backward, int64_t* bytes)
{
    if (!f || !bytes) return fail(CARL_ERR_VALUE, "null feed-forward argument");
    if (int rc = checkFfn(f, backward != 0)) return rc;
    Plan plan(f->type, nullptr);
    if (f->rows > 0) {
        if (backward) (void)Backward(*f, plan);
        else (void)Forward(*f, plan);
    }
    *bytes = plan.bytes();
    return CARL_OK;
}

int carl_gated_ffn(const carl_ffn* f, void* stream)
{
    if (int rc = checkFfn(f, false)) return rc;
    if (f->rows == 0) return CARL_OK;
    if (!f->workspace) return fail(CARL_ERR_VALUE, "null workspace");
    const hipStream_t s = (hipStream_t)stream;
    Plan plan(f->type, static_cast<char*>(f->workspace));
    const Forward p(*f, plan);
    if (f->rows <= kThinRows) {
        const ThinArgs up{ f->x, f->w_gate, f->w_up, const_cast<void*>(p.h.data), f->x_row, p.h.stride, (int32_t)f->rows, f->inner,
                           f->width, f->activation };
        if (int rc = thin(f->type, true, up, s)) return rc;
        const ThinArgs down{ p.h.data, f->w_down, nullptr, f->y, p.h.stride, f->width, (int32_t)f->rows, f->width, f->inner, 0 };
        return thin(f->type, false, down, s);
    }
    if (int rc = pack(f->type, plan.packs(), s)) return rc;
    if (int rc = scale(f->type, p.scales, s)) return rc;
    ProductArgs a{};
    a.scale[0] = factor(p.scales, kScaleH);
    a.a[0] = p.x;
    a.b[0] = p.gate;
    a.b[1] = p.up;
    a.activation = f->activation;
    a.m = f->rows;
    a.n = f->inner;
    a.out[0] = const_cast<void*>(p.h.data);
    a.outStride = p.h.stride;
    a.outWidth = p.h.width;
    a.outWide = 1;
    if (int rc = product(f->type, kProductGate, a, s)) return rc;
    ProductArgs y = toRows(*f, f->y);
    y.a[0] = p.h;
    y.b[0] = p.down;
    y.terms = 1;
    y.scale[0] = factor(p.scales, kUnscaleH);
    return product(f->type, kProductPlain, y, s);
}

int carl_gated_ffn_backward(const carl_ffn* f, void* stream)
{
    if (int rc = checkFfn(f, true)) return rc;
    const hipStream_t s = (hipStream_t)stream;
    SumArgs sum{};
    void* const weights[3] = { f->dw_gate, f->dw_up, f->dw_down };
    if (f->rows == 0) {
        for (void* w : weights)
            if (w) sum.job[sum.jobs++] = { nullptr, w, (int64_t)f->width * f->inner, nullptr };
        return sum.jobs ? sums(f->type, sum, s) : CARL_OK;
    }
    if (!f->workspace) return fail(CARL_ERR_VALUE, "null workspace");
    Plan plan(f->type, static_cast<char*>(f->workspace));
    const Backward p(*f, plan);
    if (int rc = pack(f->type, plan.packs(), s)) return rc;
    if (int rc = scale(f->type, p.scales, s)) return rc;
    ProductArgs a{};
    a.scale[0] = factor(p.scales, kScaleH);
    a.scale[1] = factor(p.scales, kScaleD);
    a.a[0] = p.x;
    a.a[1] = p.dy;
    a.b[0] = p.gate;
    a.b[1] = p.up;
    a.b[2] = p.downT;
    a.activation = f->activation;
    a.m = f->rows;
    a.n = f->inner;
    a.out[0] = const_cast<void*>(p.h.data);
    a.out[1] = const_cast<void*>(p.dg.data);
    a.out[2] = const_cast<void*>(p.du.data);
    a.outStride = p.h.stride;
    a.outWidth = p.h.width;
    a.outWide = 1;
    if (int rc = product(f->type, kProductGrad, a, s)) return rc;
    if (f->dx) {
        ProductArgs d = toRows(*f, f->dx);
        d.a[0] = p.dg;
        d.a[1] = p.du;
        d.b[0] = p.gateT;
        d.b[1] = p.upT;
        d.terms = 2;
        d.scale[0] = factor(p.scales, kUnscaleD);
        if (int rc = product(f->type, kProductPlain, d, s)) return rc;
    }
    OuterArgs outer = p.outer;
    outer.jobs = 0;
    for (int j = 0; j < 3; j++) {
        if (!weights[j]) continue;
        const int k = outer.jobs++;
        outer.p[k] = p.outer.p[j];
        outer.q[k] = p.outer.q[j];
        outer.part[k] = p.outer.part[j];
        outer.m[k] = p.outer.m[j];
        outer.n[k] = p.outer.n[j];
        sum.job[k] = { p.outer.part[j], weights[j], (int64_t)f->width * f->inner, factor(p.scales, j < 2 ? kUnscaleD : kUnscaleH) };
    }
    if (outer.jobs == 0) return CARL_OK;
    if (int rc = outerProducts(f->type, outer, p.tile, s)) return rc;
    sum.jobs = outer.jobs;
    sum.splits = outer.splits;
    return sums(f->type, sum, s);
}

}  // extern "C"
