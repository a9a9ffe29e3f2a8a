"""The C entry points of the block-scaled layer and the norm when the host has no memory left (no GPU needed): a program whose
operator new fails on demand calls each of them with arguments that are refused and with empty ones.  No exception may
leave an entry point: a refusal ends as a status, and an empty call allocates nothing."""
import os
import subprocess

from noeira_amd import _lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <dlfcn.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <new>
#include "noeira_qlinear.h"
#include "noeira_qlinear_diag.h"

static bool none_left = false;
void* operator new(size_t n) {
    void* p = none_left ? nullptr : malloc(n);
    if (!p) throw std::bad_alloc();
    return p;
}
void operator delete(void* p) noexcept { free(p); }
void operator delete(void* p, size_t) noexcept { free(p); }

static void* lib;
static int bad = 0;
#define F(name) reinterpret_cast<decltype(&name)>(dlsym(lib, #name))
#define REFUSED(call)                                                                    \
    do {                                                                                 \
        none_left = true;                                                                \
        const int rc = (call);                                                           \
        none_left = false;                                                               \
        char words[64];                                                                  \
        F(nq_last_error)(words, sizeof words);                                           \
        if (rc == NQ_OK || strcmp(words, "out of memory")) bad++, printf("%s: %d %s\n", #call, rc, words); \
    } while (0)
#define EMPTY(call)                                          \
    do {                                                     \
        none_left = true;                                    \
        const int rc = (call);                               \
        none_left = false;                                   \
        if (rc != NQ_OK) bad++, printf("%s: %d\n", #call, rc); \
    } while (0)

int main(int, char** argv) {
    lib = dlopen(argv[1], RTLD_NOW);
    if (!lib) return printf("%s\n", dlerror()), 2;
    nq_handle h = nullptr, out = nullptr;
    if (F(nq_create)(&h, NQ_FMT_FP8_BLOCK, 128, 64, 0, NQ_FLAG_GRAD)) return 3;
    void* p = reinterpret_cast<void*>(64);
    float* f = reinterpret_cast<float*>(64);
    uint8_t* c = reinterpret_cast<uint8_t*>(64);
    nq_handle two[2] = {h, h};
    void* ys[1] = {p};
    int32_t form[5];
    REFUSED(F(nq_create)(&out, NQ_FMT_FP8_BLOCK, 100, 64, 0, 0));
    REFUSED(F(nq_create)(&out, NQ_FMT_FP8_BLOCK, 128, 64, 0, 0));  // (the layer itself)
    REFUSED(F(nq_set_weight_fp8_block)(h, nullptr, nullptr, nullptr));
    REFUSED(F(nq_set_weight_fp8_block_dev)(h, nullptr, nullptr, nullptr));
    REFUSED(F(nq_forward)(h, p, NQ_DT_FP8_E4M3, f, p, NQ_DT_F32, 1, nullptr, NQ_DT_F32, NQ_EPI_NONE, nullptr));
    REFUSED(F(nq_forward_fused)(h, p, NQ_DT_FP8_E4M3, f, ys, 1, NQ_DT_F32, 1, nullptr, NQ_DT_F32, NQ_EPI_NONE, nullptr));
    REFUSED(F(nq_fuse_rows)(&out, two, 2, nullptr));
    REFUSED(F(nq_grad_input_fp8_block)(h, c, f, p, NQ_DT_F32, 1, nullptr));
    REFUSED(F(nq_quantize_rows_fp8_block)(p, NQ_DT_I8, c, f, 1, 128, nullptr));
    REFUSED(F(nq_layer_norm)(p, NQ_DT_F32, f, f, -1.0f, p, NQ_DT_F32, nullptr, nullptr, 1, 64, nullptr));
    REFUSED(F(nq_layer_norm_fp8_block)(p, NQ_DT_F32, f, f, -1.0f, c, f, nullptr, nullptr, 1, 64, nullptr));
    REFUSED(F(nq_layer_norm_grad)(p, NQ_DT_F32, f, f, f, p, NQ_DT_F32, nullptr, NQ_DT_F32, f, f, 1, 64, nullptr, 0, nullptr));
    REFUSED(F(nq_diag_fp8_block_form)(0, 1, 16, NQ_DT_F32, form));
    REFUSED(F(nq_diag_fp8_block_form)(2147483647, 64, 16, NQ_DT_F32, form));
    EMPTY(F(nq_quantize_rows_fp8_block)(p, NQ_DT_F32, c, f, 0, 128, nullptr));
    EMPTY(F(nq_layer_norm)(p, NQ_DT_F32, f, f, 1e-5f, p, NQ_DT_F32, nullptr, nullptr, 0, 64, nullptr));
    EMPTY(F(nq_layer_norm_fp8_block)(p, NQ_DT_F32, f, f, 1e-5f, c, f, nullptr, nullptr, 0, 64, nullptr));
    EMPTY(F(nq_layer_norm_grad)(p, NQ_DT_F32, f, f, f, p, NQ_DT_F32, p, NQ_DT_F32, nullptr, nullptr, 0, 64, nullptr, 0, nullptr));
    EMPTY(F(nq_diag_fp8_block_form)(100, 4096, 4096, NQ_DT_BF16, form));
    F(nq_destroy)(h);
    printf("%d\n", bad);
    return bad != 0;
}
"""


def test_no_exception_leaves_an_entry_point(tmp_path):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(PROGRAM)
    subprocess.check_call(["g++", "-std=c++17", "-rdynamic", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe), "-ldl"])
    path = next(p for p in L.candidates() if os.path.exists(p))
    r = subprocess.run([str(exe), path], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, (r.returncode, r.stdout, r.stderr)
