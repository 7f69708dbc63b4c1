/* Calls every rln_gated_* and rln_rotary_* entry point of the C ABI with arguments
 * they must refuse, and their size queries, under the host sanitizers
 * (tests/test_heads_sanitize.py). Nothing reaches a device. */
#include <math.h>
#include <stdio.h>
#include <string.h>

#include "rln.h"

#define FAKE ((void*)0x100000) /* never dereferenced */

static int failures;

static void expect(int status, const char* text, int line) {
    if (status == RLN_OK || strstr(rln_last_error(), text) == NULL) {
        fprintf(stderr, "line %d: status %d, message \"%s\" (wanted \"%s\")\n", line, status,
                rln_last_error(), text);
        ++failures;
    }
}

#define REFUSED(call, text) expect((call), (text), __LINE__)

static int gated(int64_t rows, int64_t hidden, int64_t gate_rows, int64_t weight_rows,
                 int64_t stride, double scale) {
    const rln_factor_t gate = {FAKE, RLN_DTYPE_BF16, stride, gate_rows};
    const rln_factor_t weight = {FAKE, RLN_DTYPE_F32, stride, weight_rows};
    return rln_gated_forward(FAKE, RLN_DTYPE_BF16, stride, FAKE, RLN_DTYPE_F16, stride, FAKE,
                             RLN_DTYPE_F32, &gate, &weight, FAKE, NULL, RLN_DTYPE_BF16, NULL,
                             rows, hidden, scale, 1.0, 1e-6, 1e-6, NULL);
}

static int gated_backward(int64_t rows, int64_t hidden, int64_t gate_rows, void* workspace,
                          size_t bytes) {
    const rln_factor_t gate = {FAKE, RLN_DTYPE_BF16, hidden, gate_rows};
    const rln_factor_t weight = {FAKE, RLN_DTYPE_F32, hidden, rows};
    return rln_gated_backward(NULL, FAKE, RLN_DTYPE_BF16, FAKE, RLN_DTYPE_BF16, FAKE,
                              RLN_DTYPE_F16, hidden, FAKE, RLN_DTYPE_F32, &gate, &weight, FAKE,
                              FAKE, FAKE, FAKE, FAKE, FAKE, rows, hidden, 1.0, 1.0, workspace,
                              bytes, NULL);
}

static rln_rotary_side_t side(int64_t count, int64_t stride, void* output) {
    const rln_rotary_side_t made = {{FAKE, stride, stride, stride}, {FAKE, stride, stride, stride},
                                    count, FAKE, RLN_DTYPE_F32, output, NULL};
    return made;
}

static int rotary(int64_t count, int64_t stride, int64_t outer, int64_t inner, int64_t size,
                  int64_t pairs, int64_t axes, const uint8_t* axis_of_pair) {
    const rln_rotary_side_t q = side(count, stride, NULL);
    const rln_rotary_t table = {FAKE, RLN_POSITIONS_I64, stride, stride, stride, FAKE, 0,
                                axis_of_pair, axes, pairs, 0};
    return rln_rotary_forward(&q, NULL, RLN_DTYPE_BF16, &table, outer, inner, size, 1e-6, NULL);
}

static int rotary_backward(int64_t tokens, void* workspace, size_t bytes) {
    rln_rotary_side_t q = side(8, 64, FAKE);
    const rln_rotary_t table = {FAKE, RLN_POSITIONS_F32, 0, 0, 1, FAKE, 1, NULL, 1, 32, 1};
    q.grad_weight = FAKE;
    return rln_rotary_backward(&q, NULL, RLN_DTYPE_F16, &table, 1, tokens, 64, 1e-6, workspace,
                               bytes, NULL);
}

int main(void) {
    const int64_t huge = INT64_MAX;
    const uint8_t axes[4] = {0, 1, 2, 3};
    REFUSED(gated(0, 8, 1, 1, 8, 1.0), "empty");
    REFUSED(gated(-huge - 1, 8, 1, 1, 8, 1.0), "empty");
    REFUSED(gated(huge, 8, 1, 1, 8, 1.0), "overflows");
    REFUSED(gated(4, huge, 1, 1, 8, 1.0), "hidden size");
    REFUSED(gated(4, -huge - 1, 1, 1, 8, 1.0), "hidden size");
    REFUSED(gated(4, 8, huge, 4, 8, 1.0), "gate: its rows");
    REFUSED(gated(4, 8, -huge - 1, 4, 8, 1.0), "gate: its rows");
    REFUSED(gated(4, 8, 4, 3, 8, 1.0), "weight: its rows");
    REFUSED(gated(8, 8, 2, 4, 8, 1.0), "same rows");
    REFUSED(gated(4, 8, 1, 4, huge, 1.0), "overflows");
    REFUSED(gated(4, 8, 1, 4, -huge - 1, 1.0), "overflows");
    REFUSED(gated(4, 8, 1, 4, 8, NAN), "finite");
    REFUSED(gated(4, 8, 1, 4, 8, INFINITY), "finite");
    REFUSED(gated(4, 8, 1, 4, 8, 1.0), "must not be null");
    REFUSED(gated(huge / 512, 8, 1, huge / 512, 8, 1.0), "must not be null");
    REFUSED(gated_backward(1 << 20, 8, 1 << 10, NULL, 0), "workspace too small");
    REFUSED(gated_backward((int64_t)1 << 40, 8, 2, FAKE, 1 << 20), "workspace too small");
    REFUSED(gated_backward(4, 8, 2, (char*)FAKE + 1, 1 << 20), "aligned");

    REFUSED(rotary(8, 64, 0, 4, 64, 32, 1, NULL), "empty");
    REFUSED(rotary(8, 64, huge, huge, 64, 32, 1, NULL), "number of tokens");
    REFUSED(rotary(8, 64, 2, huge, 64, 32, 1, NULL), "number of tokens");
    REFUSED(rotary(8, 64, 2, 4, huge, 32, 1, NULL), "head size");
    REFUSED(rotary(8, 64, 2, 4, 64, huge, 1, NULL), "pairs");
    REFUSED(rotary(8, 64, 2, 4, 64, -1, 1, NULL), "pairs");
    REFUSED(rotary(8, 64, 2, 4, 64, 4, 3, axes), "past the last");
    REFUSED(rotary(8, 64, 2, 4, 64, 4, huge, axes), "axes");
    REFUSED(rotary(huge, 64, 2, 4, 64, 4, 4, axes), "number of heads");
    REFUSED(rotary(-1, 64, 2, 4, 64, 4, 4, axes), "number of heads");
    REFUSED(rotary(0, 64, 2, 4, 64, 4, 4, axes), "empty");
    REFUSED(rotary(8, huge, 2, 4, 64, 4, 4, axes), "overflow");
    REFUSED(rotary(8, -huge - 1, 2, 4, 64, 4, 4, axes), "overflow");
    REFUSED(rotary(8, 64, 2, 4, 64, 4, 4, axes), "must not be null");
    REFUSED(rotary(8, huge / 64 / 8, 1, 1, 64, 4, 4, axes), "must not be null");
    REFUSED(rotary_backward(1 << 20, NULL, 0), "workspace too small");
    REFUSED(rotary_backward((1 << 30) - 1, FAKE, 256), "workspace too small");

    for (int dtype = -1; dtype <= RLN_DTYPE_INT8; ++dtype) {
        const int known = dtype >= RLN_DTYPE_F32 && dtype <= RLN_DTYPE_BF16;
        for (int64_t rows = -1; rows < (INT64_C(1) << 40); rows = rows * 7 + 9) {
            for (int64_t hidden = -1; hidden <= 20000; hidden = hidden * 2 + 3) {
                const size_t bytes =
                    rln_gated_backward_workspace_bytes(rows, hidden, dtype, rows, rows);
                const int served = known && rows > 0 && rln_rms_hidden_supported(hidden);
                if (served ? bytes == 0 || bytes > 8 * 512 * (size_t)hidden : bytes != 0) {
                    fprintf(stderr, "workspace of %lld x %lld, dtype %d: %zu\n", (long long)rows,
                            (long long)hidden, dtype, bytes);
                    ++failures;
                }
            }
            for (int64_t size = -1; size <= 300; size = size * 2 + 3) {
                for (int64_t heads = -1; heads < 100000; heads = heads * 9 + 10) {
                    const size_t bytes = rln_rotary_backward_workspace_bytes(
                        1, rows, heads, 3, size, size / 2, dtype);
                    const int served = known && rows > 0 && rows < (1 << 30) && size > 1
                        && size <= 256 && heads >= 0 && heads <= 1 << 16;
                    if (served ? bytes == 0 || bytes > 4 * 2048 * (size_t)size : bytes != 0) {
                        fprintf(stderr, "workspace of %lld tokens, %lld heads of %lld: %zu\n",
                                (long long)rows, (long long)heads, (long long)size, bytes);
                        ++failures;
                    }
                }
            }
        }
    }
    puts(failures ? "failed" : "ok");
    return failures ? 1 : 0;
}
