"""A cache whose sequences are kept on the GPU, and verification of many requests, on the host: where a page's rows lie, what is refused, and what is left behind once a call of
CUDA's runtime has failed."""
import os
import re
import subprocess

import numpy as np

from densecore_b200 import build as B
from host_util import program, run

STUBS = r"""
#include "dc_kv_dev.h"
int rows = 0, prompts = 0;
int dc_launch_kv16_rows(dc_ctx*, const dc_kv16_call&, bool) { return ++rows, 0; }
int dc_launch_kv16_prompt(dc_ctx*, const dc_kv16_call&) { return ++prompts, 0; }
size_t dc_kv16_prompt_parts(int num_sms, int n_kv, int dim) { return (size_t)num_sms * 256 * (dim + 4) * 4; }
"""


def test_every_row_has_its_place_in_a_record(tmp_path):
    """Two bytes a value, none shared; keys in the 128-byte swizzle (rows of 64 dimensions of a token, groups of eight tokens), values in the 32-byte one (rows of sixteen tokens of a
    dimension): address bits 4-6 of a linear layout xor bits 7-9, bit 4 xor bit 7."""
    src, exe = tmp_path / "p.cu", str(tmp_path / "p")
    src.write_text(r"""
#include <stdio.h>
#include "dc_kv_dev.h"
template <int HD> void all() {
    using R = dc_kv16_rec<HD>;
    for (int tok = 0; tok < 16; ++tok)
        for (int d = 0; d < HD; ++d) printf("%d %d %d %u %u %u %u\n", HD, tok, d, R::key(tok, d), R::value(tok, d), R::VALUES, R::BYTES);
}
int main() { all<64>(); all<128>(); }
""")
    subprocess.check_call([B.nvcc(), "-std=c++17", "--expt-relaxed-constexpr", "-arch=sm_100", "-I", B.CSRC, "-I", os.path.join(B.ROOT, "include"), str(src), "-o", exe])
    a = np.array([[int(x) for x in line.split()] for line in subprocess.check_output([exe], text=True).splitlines()])
    for hd in (64, 128):
        r = a[a[:, 0] == hd]
        tok, d, key, value = r[:, 1], r[:, 2], r[:, 3], r[:, 4]
        assert set(r[:, 5]) == {32 * hd} and set(r[:, 6]) == {64 * hd}
        assert sorted(key) == list(range(0, 32 * hd, 2)) and sorted(value) == list(range(32 * hd, 64 * hd, 2))
        linear = (tok // 8) * (16 * hd) + (d // 64) * 1024 + (tok % 8) * 128 + (d % 64) * 2
        assert np.array_equal(key, linear ^ ((linear >> 7 & 7) << 4))
        linear = d * 32 + tok * 2
        assert np.array_equal(value - 32 * hd, linear ^ ((linear >> 7 & 1) << 4))


def test_caches_that_are_refused_and_calls_that_fail(tmp_path):
    """Shapes beyond what is supported allocate nothing; a cache that fails to be made at any call leaves nothing behind."""
    exe = program(tmp_path, ["kv_dev", "kv"], STUBS + r"""
int main() {
    dc_ctx ctx;
    dc_kv_cache* kv = nullptr;
    const int F16 = DC_GGML_TYPE_F16, bad[][9] = {      // layers, heads, key heads, size, type, pages, sequences, pages a sequence, tokens
        {0, 8, 2, 64, F16, 9, 2, 3, 4}, {1, 0, 2, 64, F16, 9, 2, 3, 4}, {1, 8, 0, 64, F16, 9, 2, 3, 4}, {1, 8, 3, 64, F16, 9, 2, 3, 4}, {1, 8, 2, 96, F16, 9, 2, 3, 4}, {1, 8, 2, 256, F16, 9, 2, 3, 4},
        {1, 8, 2, 64, DC_GGML_TYPE_Q4_K, 9, 2, 3, 4}, {1, 8, 2, 64, F16, 0, 2, 3, 4}, {1, 8, 2, 64, F16, 9, 0, 3, 4}, {1, 8, 2, 64, F16, 9, 4097, 3, 4}, {1, 8, 2, 64, F16, 9, 2, 0, 4},
        {1, 8, 2, 64, F16, 9, 4000, 1 << 20, 4}, {1, 8, 2, 64, F16, 9, 2, 1 << 27, 4}, {1, 8, 2, 64, F16, 9, 2, 3, 0}, {1, 8, 2, 64, F16, 9, 2, 3, 1 << 28}, {1, 8, 2, 64, F16, (1 << 26) + 1, 2, 3, 4},
        {2147483647, 65536, 65535, 128, F16, 1 << 26, 2, 3, 4}, {-1, -8, -2, -64, F16, -9, -2, -3, -4}};
    for (auto& b : bad) {
        const int st = dc_b200_kv_create_dev(&ctx, b[0], b[1], b[2], b[3], b[4], b[5], b[6], b[7], b[8], &kv);
        if ((st != DC_B200_INVALID_ARGUMENT && st != DC_B200_UNSUPPORTED) || kv || fake::calls) return printf("%d heads, %d pages: status %d\n", b[1], b[5], st), 1;
    }
    if (dc_b200_kv_create_dev(&ctx, 1, 8, 2, 64, F16, 9, 2, 3, 4, nullptr) != DC_B200_INVALID_ARGUMENT) return printf("no place for the cache\n"), 1;
    for (int n = 1;; ++n) {
        fake::calls = 0, fake::fail_at = n;
        const int st = dc_b200_kv_create_dev(&ctx, 3, 8, 2, 64, DC_GGML_TYPE_BF16, 60, 4, 40, 100, &kv);
        const bool failed = fake::calls >= n;
        if (failed != (st != 0) || failed != !kv) return printf("call %d: status %d\n", n, st), 1;
        dc_b200_kv_destroy(kv);
        if (fake::bad_frees || !fake::live.empty()) return printf("call %d: %d freed twice, %d lost\n", n, fake::bad_frees, (int)fake::live.size()), 1;
        if (!failed) return printf("%d calls\n", n - 1), 0;
    }
}
""")
    r = run(exe)
    assert r.returncode == 0 and int(r.stdout.split()[0]) >= 6, r.stdout


def test_calls_that_are_refused_launch_nothing(tmp_path):
    """Caches of other kinds, of another context, before a first step, layers, strides, masks, alignments; and which kernels the allowed ones launch."""
    exe = program(tmp_path, ["kv_dev", "kv"], STUBS + r"""
int main() {
    dc_ctx ctx, other;
    dc_kv_cache *kv = nullptr, *plain = nullptr, *f32 = nullptr;
    char* x = (char*)(size_t(1) << 40);      // (nothing reads them here)
    if (dc_b200_kv_create_dev(&ctx, 2, 16, 2, 64, DC_GGML_TYPE_BF16, 60, 4, 40, 1000, &kv) || dc_b200_kv_create_dev(&ctx, 2, 16, 2, 64, DC_GGML_TYPE_F32, 60, 4, 40, 1000, &f32)) return printf("create\n"), 1;
    if (dc_b200_kv_create(&ctx, 1, 2, 128, 9, 2, 4, &plain)) return printf("a plain one\n"), 1;
    int seq = -1, n = 0;
    dc_kv_dev_arrays a;
    auto attend = [&](dc_ctx* c, dc_kv_cache* z, int layer, const void* q, int64_t ldq, const void* k, const void* v, int64_t ldk, float scale, int window, int keep, void* out, int64_t ldo) {
        return dc_b200_flash_attn_kv_dev(c, z, layer, q, ldq, k, v, ldk, scale, window, keep, out, ldo);
    };
    fake::launches = 0;
    const float nan = 0.0f / 0.0f * 1.0f;
    struct { const char* what; int st; } early[] = {
        {"before a step", attend(&ctx, kv, 0, x, 0, x, x, 0, 1, 0, 0, x, 0)}, {"rows before a step", dc_b200_kv_dev_write_dev(&ctx, kv, 0, x, x, 0)},
        {"another kind", attend(&ctx, plain, 0, x, 0, x, x, 0, 1, 0, 0, x, 0)}, {"its step", dc_b200_kv_step_dev(&ctx, plain, nullptr, nullptr, 1)}, {"its arrays", dc_b200_kv_dev_arrays(plain, &a)},
        {"its page", dc_b200_kv_dev_read_page(plain, 0, 0, nullptr, nullptr)}, {"another context", dc_b200_kv_step_dev(&other, kv, nullptr, nullptr, 1)}, {"a negative limit", dc_b200_kv_step_dev(&ctx, kv, nullptr, nullptr, -1)},
        {"no cache", dc_b200_kv_step_dev(&ctx, nullptr, nullptr, nullptr, 1)}, {"no context", dc_b200_kv_step_dev(nullptr, kv, nullptr, nullptr, 1)}, {"a sequence", dc_b200_kv_seq_alloc(kv, &seq)},
        {"a reservation", dc_b200_kv_seq_reserve(kv, 0, 4)}, {"a fork", dc_b200_kv_seq_fork(kv, 0, &seq)}, {"a table", dc_b200_kv_block_table(kv, 0, nullptr, 0, &n)}, {"free blocks", dc_b200_kv_free_blocks(kv)},
        {"a prefix", dc_b200_kv_prefix_attach(kv, 0, &n, 1, &seq)}, {"a block", dc_b200_kv_read_block(kv, 0, 0, nullptr, nullptr)}, {"a page behind", dc_b200_kv_dev_read_page(kv, 0, 60, nullptr, nullptr)}};
    for (auto& e : early)
        if (e.st >= 0 || fake::launches || rows) return printf("%s: status %d\n", e.what, e.st), 1;
    if (dc_b200_kv_step_dev(&ctx, kv, nullptr, nullptr, 1) || fake::launches != 1) return printf("a step\n"), 1;
    struct { const char* what; int st; } late[] = {
        {"layer", attend(&ctx, kv, 2, x, 0, x, x, 0, 1, 0, 0, x, 0)}, {"layer below 0", attend(&ctx, kv, -1, x, 0, x, x, 0, 1, 0, 0, x, 0)}, {"no queries", attend(&ctx, kv, 0, nullptr, 0, x, x, 0, 1, 0, 0, x, 0)},
        {"no results", attend(&ctx, kv, 0, x, 0, x, x, 0, 1, 0, 0, nullptr, 0)}, {"keys alone", attend(&ctx, kv, 0, x, 0, x, nullptr, 0, 1, 0, 0, x, 0)}, {"values alone", attend(&ctx, kv, 0, x, 0, nullptr, x, 0, 1, 0, 0, x, 0)},
        {"short rows", attend(&ctx, kv, 0, x, 1023, x, x, 0, 1, 0, 0, x, 0)}, {"short key rows", attend(&ctx, kv, 0, x, 0, x, x, 127, 1, 0, 0, x, 0)}, {"short result rows", attend(&ctx, kv, 0, x, 0, x, x, 0, 1, 0, 0, x, -5)},
        {"scale", attend(&ctx, kv, 0, x, 0, x, x, 0, nan, 0, 0, x, 0)}, {"infinite scale", attend(&ctx, kv, 0, x, 0, x, x, 0, 1e39f, 0, 0, x, 0)}, {"window", attend(&ctx, kv, 0, x, 0, x, x, 0, 1, -1, 0, x, 0)},
        {"kept", attend(&ctx, kv, 0, x, 0, x, x, 0, 1, 5, -1, x, 0)}, {"kept without a window", attend(&ctx, kv, 0, x, 0, x, x, 0, 1, 0, 4, x, 0)}, {"an odd address", attend(&ctx, kv, 0, x + 1, 0, x, x, 0, 1, 0, 0, x, 0)},
        {"an odd result", attend(&ctx, kv, 0, x, 0, x, x, 0, 1, 0, 0, x + 3, 0)}, {"f32 off its size", (dc_b200_kv_step_dev(&ctx, f32, nullptr, nullptr, 1), attend(&ctx, f32, 0, x + 2, 0, x, x, 0, 1, 0, 0, x, 0))},
        {"no rows", dc_b200_kv_dev_write_dev(&ctx, kv, 0, nullptr, x, 0)}, {"rows of another layer", dc_b200_kv_dev_write_dev(&ctx, kv, 7, x, x, 0)}, {"short written rows", dc_b200_kv_dev_write_dev(&ctx, kv, 0, x, x, 5)}};
    for (auto& e : late)
        if (e.st >= 0 || rows || prompts) return printf("%s: status %d\n", e.what, e.st), 1;
    // eight rows a token: 8 tokens are the rows kernel's, 9 bring the prompts' and the writing one; f32 rows of 5 tokens the rows kernel twice
    struct { dc_kv_cache* z; int most, launches, rows, prompts; } runs[] = {{kv, 0, 0, 0, 0}, {kv, 8, 0, 1, 0}, {kv, 9, 1, 1, 1}, {f32, 4, 0, 1, 0}, {f32, 5, 1, 2, 0}};
    for (auto& r : runs) {
        dc_b200_kv_step_dev(&ctx, r.z, nullptr, nullptr, r.most);
        fake::launches = rows = prompts = 0;
        if (attend(&ctx, r.z, 1, x, 0, x, x, 0, 1, 3, 1, x, 0) || fake::launches != r.launches || rows != r.rows || prompts != r.prompts) return printf("%d tokens: %d %d %d\n", r.most, fake::launches, rows, prompts), 1;
    }
    dc_b200_kv_destroy(kv), dc_b200_kv_destroy(f32), dc_b200_kv_destroy(plain);
    return fake::bad_frees || !fake::live.empty();
}
""")
    r = run(exe)
    assert r.returncode == 0, r.stdout


def test_verifications_that_are_refused(tmp_path):
    """Shapes, types and buffers; a first call within a capture; a workspace that cannot be had."""
    exe = program(tmp_path, ["verify_rows"], r"""
int main() {
    dc_ctx ctx;
    char* x = (char*)(size_t(1) << 40);
    const int F32 = DC_GGML_TYPE_F32;
    auto call = [&](const void* target, int type, int64_t ld, int rows, int V, int R, int D, const void* tokens, const void* u, void* out, void* acc) {
        return dc_b200_verify_rows_dev(&ctx, target, type, ld, rows, V, R, D, nullptr, nullptr, (const int*)tokens, nullptr, nullptr, (const float*)u, (int*)out, (int*)acc, nullptr);
    };
    struct { const char* what; int st; } bad[] = {
        {"no logits", call(nullptr, F32, 0, 8, 9, 2, 3, x, x, x, x)}, {"no tokens", call(x, F32, 0, 8, 9, 2, 3, nullptr, x, x, x)}, {"no numbers", call(x, F32, 0, 8, 9, 2, 3, x, nullptr, x, x)},
        {"no results", call(x, F32, 0, 8, 9, 2, 3, x, x, nullptr, x)}, {"no counts", call(x, F32, 0, 8, 9, 2, 3, x, x, x, nullptr)}, {"type", call(x, DC_GGML_TYPE_F16, 0, 8, 9, 2, 3, x, x, x, x)},
        {"short rows", call(x, F32, 8, 8, 9, 2, 3, x, x, x, x)}, {"no vocabulary", call(x, F32, 0, 8, 0, 2, 3, x, x, x, x)}, {"a large one", call(x, F32, 0, 8, 389121, 2, 3, x, x, x, x)}, {"drafts", call(x, F32, 0, 8, 9, 2, 65, x, x, x, x)},
        {"negative drafts", call(x, F32, 0, 8, 9, 2, -1, x, x, x, x)}, {"rows in all", call(x, F32, 0, 8, 9, 16385, 3, x, x, x, x)}, {"negative requests", call(x, F32, 0, 8, 9, -1, 3, x, x, x, x)},
        {"negative rows", call(x, F32, 0, -1, 9, 2, 3, x, x, x, x)}, {"alignment", call(x + 2, F32, 0, 8, 9, 2, 3, x, x, x, x)}};
    for (auto& b : bad)
        if (b.st >= 0 || fake::launches || fake::calls) return printf("%s: status %d\n", b.what, b.st), 1;
    if (call(x, F32, 0, 8, 9, 0, 3, x, x, x, x) || fake::launches) return printf("no requests\n"), 1;
    fake::capturing = true;
    if (call(x, F32, 0, 8, 9, 2, 3, x, x, x, x) != DC_B200_UNSUPPORTED || fake::launches) return printf("captured first\n"), 1;
    fake::capturing = false;
    for (int n = 1; n <= 2; ++n) {
        fake::calls = 0, fake::fail_at = n;
        if (call(x, F32, 0, 8, 9, 2, 3, x, x, x, x) >= 0 || fake::launches || !fake::live.empty()) return printf("failing call %d\n", n), 1;
    }
    fake::fail_at = 0, fake::capturing = false;
    if (call(x, F32, 0, 8, 9, 2, 3, x, x, x, x) || fake::launches != 2 || fake::live.size() != 1) return printf("two requests\n"), 1;
    fake::capturing = true;
    if (call(x, DC_GGML_TYPE_BF16, 0, 64 * 65, 389120, 64, 64, x, x, x, x) || fake::launches != 4 || fake::live.size() != 1) return printf("captured\n"), 1;
    if (call(x, -1, 0, 8, 9, 2, 3, x, x, x, x) || fake::launches != 5) return printf("probabilities\n"), 1;
    if (call(x, F32, 0, 8, 9, 2, 0, nullptr, x, x, x) || fake::launches != 7) return printf("no drafts\n"), 1;
    return 0;
}
""")
    r = run(exe)
    assert r.returncode == 0, r.stdout


def test_the_prompt_kernel_does_not_spill(tmp_path):
    """It loads from tensor memory: its launcher refuses a build with any local memory."""
    path = os.path.join(B.CSRC, "attn_kv16_prompt.cu")
    cmd = [B.nvcc(), "-Xptxas", "-v", *B.NVCC_FLAGS, "-I", os.path.join(B.ROOT, "include"), "-c", path, "-o", str(tmp_path / "o.o")]
    out = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, check=True).stdout
    bodies = [body for name, body in re.findall(r"Compiling entry function '(\w+)'(.*?)(?=Compiling entry|\Z)", out, re.S) if "k_kv16_prompt" in name]
    assert len(bodies) == 4 and all("0 bytes stack frame, 0 bytes spill stores, 0 bytes spill loads" in b for b in bodies)
