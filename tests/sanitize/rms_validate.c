/* Calls every rln_rms_* entry point and rln_dequantize of the C ABI with
 * arguments they must refuse, and their size queries, under the host
 * sanitizers (tests/test_rms_sanitize.py). Nothing reaches a device. */
#include <math.h>
#include <stdio.h>
#include <string.h>

#include "rln.h"

#define FAKE ((void*)0x100000) /* never dereferenced */

static int failures;

static void expect(int status, int wanted, const char* text, int line) {
    if (status != wanted || strstr(rln_last_error(), text) == NULL) {
        fprintf(stderr, "line %d: status %d (wanted %d), message \"%s\" (wanted \"%s\")\n", line,
                status, wanted, rln_last_error(), text);
        ++failures;
    }
}

#define REFUSED(call, text) expect((call), RLN_ERR_INVALID, (text), __LINE__)
#define UNSUPPORTED(call, text) expect((call), RLN_ERR_UNSUPPORTED, (text), __LINE__)

static int forward(void* x, int x_dtype, int64_t stride, void* branch, void* updated,
                   void* normalized, int8_t* checkpoint, int64_t rows, int64_t hidden,
                   double eps) {
    return rln_rms_forward(x, x_dtype, stride, branch, RLN_DTYPE_F16, stride, FAKE, RLN_DTYPE_F32,
                           updated, normalized, RLN_DTYPE_BF16, NULL, checkpoint, NULL, rows,
                           hidden, eps, NULL);
}

static int quantize(int dtype, int64_t group, float* scale, int64_t rows, int64_t hidden) {
    return rln_rms_quantize(FAKE, RLN_DTYPE_BF16, hidden, NULL, 0, 0, FAKE, RLN_DTYPE_BF16, NULL,
                            FAKE, dtype, scale, group, rows, hidden, 1e-6, NULL);
}

static int backward(void* updated, int8_t* checkpoint, void* grad_weight, void* workspace,
                    size_t bytes, int64_t rows, int64_t hidden) {
    return rln_rms_backward(NULL, FAKE, RLN_DTYPE_BF16, updated, hidden, checkpoint, NULL,
                            RLN_DTYPE_BF16, FAKE, RLN_DTYPE_BF16, FAKE, FAKE, NULL, 0, grad_weight,
                            rows, hidden, workspace, bytes, NULL);
}

static int dequantize(int dtype, int64_t group, void* values, int64_t rows, int64_t hidden) {
    return rln_dequantize(FAKE, dtype, FAKE, group, values, RLN_DTYPE_F16, rows, hidden, NULL);
}

int main(void) {
    const int64_t huge = INT64_MAX;
    REFUSED(forward(FAKE, 0, 8, FAKE, FAKE, FAKE, NULL, 0, 8, 1e-6), "empty");
    REFUSED(forward(FAKE, 0, 8, FAKE, FAKE, FAKE, NULL, -huge, 8, 1e-6), "empty");
    REFUSED(forward(FAKE, 0, 8, FAKE, FAKE, FAKE, NULL, huge, 8, 1e-6), "overflows");
    UNSUPPORTED(forward(FAKE, 0, 8, FAKE, FAKE, FAKE, NULL, 4, 0, 1e-6), "hidden size");
    UNSUPPORTED(forward(FAKE, 0, 8, FAKE, FAKE, FAKE, NULL, 4, huge, 1e-6), "hidden size");
    UNSUPPORTED(forward(FAKE, 0, 8, FAKE, FAKE, FAKE, NULL, 4, -huge - 1, 1e-6), "hidden size");
    REFUSED(forward(FAKE, 0, huge, FAKE, FAKE, FAKE, NULL, 4, 8, 1e-6), "stride overflows");
    REFUSED(forward(FAKE, 0, -huge - 1, FAKE, FAKE, FAKE, NULL, 4, 8, 1e-6), "stride overflows");
    REFUSED(forward(FAKE, -7, 8, FAKE, FAKE, FAKE, NULL, 4, 8, 1e-6), "x must use");
    REFUSED(forward(NULL, 0, 8, FAKE, FAKE, FAKE, NULL, 4, 8, 1e-6), "must not be null");
    REFUSED(forward(FAKE, 0, 8, NULL, FAKE, FAKE, NULL, 4, 8, 1e-6), "both be");
    REFUSED(forward(FAKE, 0, 8, FAKE, NULL, FAKE, NULL, 4, 8, 1e-6), "both be");
    REFUSED(forward(FAKE, 0, 8, FAKE, FAKE, NULL, NULL, 4, 8, 1e-6), "must not be null");
    REFUSED(forward(FAKE, 0, 8, FAKE, FAKE, FAKE, FAKE, 4, 8, 1e-6), "checkpoint_scale must both");
    REFUSED(forward(FAKE, 0, 8, FAKE, FAKE, FAKE, NULL, 4, 8, -1.0), "eps");
    REFUSED(forward(FAKE, 0, 8, FAKE, FAKE, FAKE, NULL, 4, 8, NAN), "eps");
    REFUSED(forward((char*)FAKE + 2, 0, 8, FAKE, FAKE, FAKE, NULL, 4, 8, 1e-6), "aligned");

    REFUSED(quantize(RLN_DTYPE_BF16, 0, FAKE, 4, 8), "quantized must use");
    REFUSED(quantize(RLN_DTYPE_INT8, 33, FAKE, 4, 8), "group must be");
    REFUSED(quantize(RLN_DTYPE_INT8, -huge - 1, FAKE, 4, 8), "group must be");
    REFUSED(quantize(RLN_DTYPE_E4M3, 128, NULL, 4, 8), "must not be null");
    REFUSED(quantize(RLN_DTYPE_E4M3, 128, FAKE, huge, 8), "overflows");

    REFUSED(backward(FAKE, NULL, NULL, NULL, 0, 0, 8), "empty");
    UNSUPPORTED(backward(FAKE, NULL, NULL, NULL, 0, 4, 16385), "hidden size");
    REFUSED(backward(NULL, NULL, NULL, NULL, 0, 4, 8), "either updated");
    REFUSED(backward(NULL, FAKE, NULL, NULL, 0, 4, 8), "either updated");
    REFUSED(backward(FAKE, NULL, FAKE, NULL, 0, 1 << 24, 8), "workspace too small");
    REFUSED(backward(FAKE, NULL, FAKE, FAKE, 31, 1 << 24, 8), "workspace too small");
    REFUSED(backward(FAKE, NULL, FAKE, FAKE, 31, huge / 64, 8), "workspace too small");
    REFUSED(backward(FAKE, NULL, FAKE, (char*)FAKE + 1, 4096, 4, 8), "aligned");

    REFUSED(dequantize(RLN_DTYPE_INT8, 0, FAKE, 0, 8), "empty");
    REFUSED(dequantize(RLN_DTYPE_INT8, 0, FAKE, 4, -1), "empty");
    UNSUPPORTED(dequantize(RLN_DTYPE_INT8, 0, FAKE, 4, huge), "row length");
    REFUSED(dequantize(RLN_DTYPE_INT8, 0, FAKE, huge, 1 << 30), "overflows");
    REFUSED(dequantize(RLN_DTYPE_F32, 0, FAKE, 4, 8), "quantized must use");
    REFUSED(dequantize(RLN_DTYPE_INT8, 7, FAKE, 4, 8), "group must be");
    REFUSED(dequantize(RLN_DTYPE_INT8, 0, NULL, 4, 8), "must not be null");

    for (int dtype = -1; dtype <= RLN_DTYPE_E4M3; ++dtype) {
        for (int64_t rows = -1; rows < (INT64_C(1) << 40); rows = rows * 7 + 9) {
            for (int64_t hidden = -1; hidden <= 20000; hidden = hidden * 2 + 3) {
                const size_t bytes = rln_rms_backward_workspace_bytes(rows, hidden, dtype);
                const int served = rows > 0 && rln_rms_hidden_supported(hidden)
                    && dtype >= RLN_DTYPE_F32 && dtype <= RLN_DTYPE_BF16;
                /* none for launches of at most 1024 rows and 2^21 elements */
                const int wanted =
                    served && (rows > 1024 || rows * hidden > (int64_t)1 << 21);
                if (wanted ? bytes == 0 || bytes > 4 * 512 * (size_t)hidden : bytes != 0) {
                    fprintf(stderr, "workspace of %lld x %lld, dtype %d: %zu\n", (long long)rows,
                            (long long)hidden, dtype, bytes);
                    ++failures;
                }
            }
        }
    }
    if (rln_rms_backward_workspace_bytes(huge, 16384, RLN_DTYPE_F32) > ((size_t)1 << 30)) {
        ++failures;
    }
    puts(failures ? "failed" : "ok");
    return failures ? 1 : 0;
}
