// attention.h - linear attention with a decay for each head, chunked form.
//
// One kernel runs every direction.  With queries a, keys b and values c,
//   out_t = sum over s of w(t, s) (a_t . b_s) c_s        (+ carried memory)
// is the forward pass for (q, k, v), and each gradient is the same sum with
// the roles exchanged: dq from (dout, v, k), and, with time running backwards
// (s >= t), dk from (v, dout, q) and dv from (k, q, dout).  w(t, s) is
// decay^|t-s| where no episode starts between the two steps, else 0.
//
// In chunks of kC steps, with X the chunk's rows and M the memory before it:
//   P = (A B^T) o w          [kC x kC]
//   out = P C + w_in A M     w_in(t) = decay^(steps since the chunk's edge)
//   M  <- w_all M + B^T (w_out C)
// Products run on the matrix cores as 16x16 tiles, k in groups of 16: a lane's
// fragment of either operand is row or column lane%16 and k = 4 (lane/16) + j,
// and its share of a result is column lane%16, rows 4 (lane/16) + i.  So the
// transposed tile P^T leaves a lane four neighbouring s of one t, and the
// memory's tile (rows: a's dimension, column: c's) is, as it stands, the
// operand M^T of the next chunk: it never leaves the registers.  Each wave
// owns 16-column tiles of c, all rows.
//
// Precision with bfloat16 rows: P is rounded once, and so is the memory where a
// reads it (each the error of one rounding of its part of the output).  w_out C
// meets B as terms of bfloat16: three where the memory is handed to the caller,
// which keeps that within float32's error of sums, else two (2^-16 of each
// addend, little beside the rounding that follows).  float16's range holds
// neither P nor the memory nor such terms: all its products but A B^T run in
// float32, and only outputs are rounded.
//
// What bounds it: no unit throughout, but the chain from a chunk's copies over
// P to its outputs, which only other workgroups of the compute unit hide.
// 16,384 x 64 steps, 8 heads of 64 in bfloat16: forward 2.26 ms (8.6 GB, 3.8
// TB/s), gradients 4.2 ms (11.8 GB, 2.8 TB/s), four workgroups a compute unit;
// in float16, most of whose products run on the float32 instructions, 2.47 and
// 6.4 ms.  6 x 4,603 steps, 8 heads of 128 on 4: 88 and 316 us for the outputs'
// and the gradients' launch, two workgroups a compute unit, matrix cores busy 10%.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/carl_amd_ops.h"
#include "elem.h"

namespace carl {

struct Rows {
    void* data;
    int64_t batch, step, head;
};

// One direction of one pass.
struct Role {
    Rows a, b, c, out;
    int32_t aHeads, bHeads, cHeads;         // query heads that share a row of each
    int32_t aGrain, bGrain, cGrain;         // bytes that its rows' addresses and widths are multiples of: 16, 8, 4 or 2
                                            // (0 where a chunk's rows do not lie within 32 bits)
    int32_t outWide;                        // out's rows take stores of four elements, and are whole ones
    int32_t outFloat;                       // out is float32 whatever the rows' type
    int32_t dimA, dimC;
    int32_t backwards;
    int32_t inShift;                        // steps between the memory before a chunk and its first row (1; backwards 0,
                                            // where the memory is the gradient of the one at the chunk's last step)
    float scaleP, scaleIn, scaleOut;        // of P, of the carried memory where it is read, of what enters the memory
    const float* first;                     // the memory before the first chunk, or NULL
    float* last;                            // after the last one, or NULL
    int32_t firstSwapped, lastSwapped;      // stored as [dimC, dimA]
    float* parts;                           // split passes: [segment, batch, head, dimA, dimC] and a factor for each
    float* factors;
    int32_t partsSwapped;                   // read from the parts of a role whose memory is this one's transpose
};

struct Pass {
    Role role[3];
    int64_t batch, steps;
    int32_t heads, segments;
    int32_t finer;                          // memories in the parts for each segment: those that its parts leave
    int32_t dealGroups;                     // whole sequences (or segments) are dealt to the dies, else heads are
    int64_t segmentSteps;
    const float* logDecay;
    const uint8_t* starts;
    int64_t startsBatch, startsStep;
};

// kStates: only the memories that the segments leave, each from zero.
int launchAttention(int type, const Pass& pass, int firstRole, int roles, bool states, hipStream_t stream);

template <typename T> int launchAttentionOf(const Pass& pass, int firstRole, int roles, bool states, hipStream_t stream);

}  // namespace carl
