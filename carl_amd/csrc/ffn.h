// ffn.h - the gated feed-forward block's products on the matrix cores.
//
//   h = act(x Wg^T) o (x Wu^T)          y = h Wd^T
//   dh = dy Wd      dg = dh o up o act'(gate)      du = dh o act(gate)
//   dx = dg Wg + du Wu      dWg = dg^T x      dWu = du^T x      dWd = dy^T h
// act(g) = g s(z(g)) with s the logistic function and z = g (SiLU) or
// z = 2 sqrt(2/pi) (g + 0.044715 g^3) (GELU in its tanh form, since
// (1 + tanh u) / 2 = s(2u)); act'(g) = s + g s (1 - s) z'(g).
//
// The backward pass recomputes gate and up in the kernel that forms dh, beside
// it: nothing is kept between the passes, and dg, du and h come from float32
// values with one rounding each (kept in 16 bits they would be rounded twice).
// Kept in 32 bits they would be 16 bytes written and read an element against
// 4 D operations: more time than the operations take up to a width of about
// 700 in 16 bits, but only up to about 100 in float32 (62,000 x 256 x 683: an
// estimated 140 us for the bytes, 390 for the second run).
//
// float16's range holds neither any h, dg and du nor the bits of small ones:
// they are written times a power of two, the same for all rows, and the
// products that read them undo it.  |act(g)| <= |g| and norms bound what they
// can be:
//   |h| <= |x| |Wg| |x| |Wu|      |dg|, |du| <= 1.13 |dy| |Wd| |x| max(|Wg|, |Wu|)
// with the largest norm of a row of x and dy, of a row of Wg and Wu and of a
// column of Wd each (rows that are not finite aside: what they give is not
// either).  The bound goes to 2^15 at most, so that nothing overflows and 29
// powers of two below keep all their bits.
//
// Three kernels do all products.  `product` multiplies rows by rows (both
// operands contiguous along the sum); `outer` sums over rows (both operands
// contiguous across it), for the weights' gradients.  Both copy panels (of 64
// or 128 bytes a row along the sum, of 32 or 64 rows across it) straight into
// LDS, two stages, one barrier a stage.  `thin` is the forward pass of up to
// 128 rows, from memory to registers.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/carl_amd_ops.h"
#include "elem.h"

namespace carl {

struct Panel {
    const void* data;      // 16-byte aligned, rows of `stride` elements, a multiple of 16 bytes
    int64_t rows, stride;
    int32_t width;         // elements along a row that count, rounded up to 16 bytes (the rest are zero)
};

enum { kProductPlain = 0, kProductGate = 1, kProductGrad = 2 };

struct ProductArgs {
    Panel a[2], b[3];      // plain: the sum of a[i] b[i]^T; gate: a[0] with b[0], b[1]; grad: those, and a[1] with b[2]
    int32_t terms;
    int32_t activation;
    int64_t m;
    int32_t n;
    void* out[3];          // plain: out; gate: h; grad: h, dg, du
    int64_t outStride;
    int32_t outWidth;      // columns that are written (gate, grad: to the end of the padding)
    int32_t outWide;       // rows are 16-byte aligned
    const float* scale[2]; // float16: factors of out[0] and of the others
};

// The forward pass of a few rows: operands as they lie, whatever their addresses.
struct ThinArgs {
    const void* a;                // [m, k], rows aStride apart: x, or h
    const void *b0, *b1;          // [n, k]; b1 for gate
    void* out;                    // [m, n], rows outStride apart: h (of up to 16 rows, or of float16, in float32), or y
    int64_t aStride, outStride;
    int32_t m, n, k, activation;
};

struct OuterArgs {
    Panel p[3], q[3];      // part[f][d] = sum over rows of p[row][f] q[row][d]
    float* part[3];        // [split][m][n]
    int32_t m[3], n[3];
    int64_t k;             // rows
    int64_t splitRows;     // of a split, a multiple of the stage
    int32_t splits, jobs;
};

struct PackJob {
    const void* from;
    void* to;
    int64_t rows, cols, fromStride, toStride;   // to: rows x toStride, zero past cols (transposed: cols x toStride, past rows)
    int32_t transposed;
};

struct PackArgs {
    PackJob job[8];
    int32_t jobs;
};

struct SumJob {
    const float* part;
    void* out;
    int64_t count;
    const float* scale;    // float16: a factor of the sum, or NULL for none
};

struct SumArgs {
    SumJob job[3];
    int32_t splits, jobs;
};

// The largest rows by their norm, of x, w_gate, w_up and, backwards, of dy and
// of w_down's transpose, and from them the factors of h and of dg and du.
struct ScaleArgs {
    Panel rows[5];
    float* part;           // [5][kScaleBlocks]
    float* scale;          // of h, of dg and du, and what undoes each
    int32_t panels;        // 3 or 5
};
constexpr int kScaleBlocks = 2048;
enum { kScaleH = 0, kScaleD = 1, kUnscaleH = 2, kUnscaleD = 3 };

int launchScale(const ScaleArgs& args, hipStream_t stream);      // float16

template <typename T> int launchProduct(int kind, const ProductArgs& args, hipStream_t stream);
template <typename T> int launchThin(bool gate, const ThinArgs& args, hipStream_t stream);
template <typename T> int launchOuter(const OuterArgs& args, int tile, hipStream_t stream);
template <typename T> int launchPack(const PackArgs& args, hipStream_t stream);
template <typename T> int launchSum(const SumArgs& args, hipStream_t stream);

// Columns and rows of an outer product's tile for these sizes.
int outerTile(int m, int n);

}  // namespace carl
