"""Buffers of the calls of steps on the GPU that no kernel may be given: numbers off their own size, and results in the place of what the call's CTAs still read."""
from host_util import program, run
from test_kv_dev_cpu import STUBS


def test_step_numbers_off_their_size(tmp_path):
    exe = program(tmp_path, ["kv_dev", "kv"], STUBS + r"""
int main() {
    dc_ctx ctx;
    dc_kv_cache* kv = nullptr;
    char* x = (char*)(size_t(1) << 40);      // (nothing reads it here)
    auto at = [&](int n) { return (const int32_t*)(x + n); };
    if (dc_b200_kv_create_dev(&ctx, 1, 8, 2, 64, DC_GGML_TYPE_BF16, 60, 4, 40, 100, &kv)) return printf("create\n"), 1;
    fake::launches = 0;
    for (int n = 1; n < 4; ++n)
        if (dc_b200_kv_step_dev(&ctx, kv, at(n), at(0), 3) != DC_B200_INVALID_ARGUMENT || dc_b200_kv_step_dev(&ctx, kv, nullptr, at(n), 3) != DC_B200_INVALID_ARGUMENT || fake::launches) return printf("off by %d\n", n), 1;
    if (dc_b200_flash_attn_kv_dev(&ctx, kv, 0, x, 0, x, x, 0, 1, 0, 0, x, 0) >= 0) return printf("a refused step counts\n"), 1;
    if (dc_b200_kv_step_dev(&ctx, kv, at(4), at(8), 3) || fake::launches != 1) return printf("aligned ones\n"), 1;
    dc_b200_kv_destroy(kv);
    return fake::bad_frees || !fake::live.empty();
}
""")
    r = run(exe)
    assert r.returncode == 0, r.stdout


def test_verification_buffers(tmp_path):
    exe = program(tmp_path, ["verify_rows"], r"""
int main() {
    dc_ctx ctx;
    char* x = (char*)(size_t(1) << 40);
    // target, draft probabilities, starts, numbers of drafts, draft tokens, temperatures, uniform numbers, tokens, accepted, rejected: a megabyte apart
    auto call = [&](int which, long off) {
        const char* a[10];
        for (int i = 0; i < 10; ++i) a[i] = x + ((long)i << 20) + (i == which ? off : 0);
        return dc_b200_verify_rows_dev(&ctx, a[0], DC_GGML_TYPE_F32, 0, 40, 50, 10, 3, (const int*)a[2], (const int*)a[3], (const int*)a[4], (const float*)a[1], (const float*)a[5], (const float*)a[6],
                                       (int*)a[7], (int*)a[8], (int*)a[9]);
    };
    for (int i = 0; i < 10; ++i)
        for (int off = 1; off < 4; ++off)
            if (call(i, off) != DC_B200_INVALID_ARGUMENT || fake::launches || fake::calls) return printf("buffer %d off by %d\n", i, off), 1;
    // ten requests' numbers are 40 bytes: results in, across and just beside those of starts, drafts and temperatures (buffers 2, 3, 5), rejected ones of the other results too
    for (int result = 7; result < 10; ++result)
        for (int other : {2, 3, 5, 7, 8, 9}) {
            if (other >= 7 && (result != 9) == (other != 9)) continue;
            const long to = ((long)(other - result) << 20), size = result == 7 ? 160 : 40, others = other == 7 ? 160 : 40;
            for (long d : {0L, 36L, -36L})
                if (call(result, to + d) != DC_B200_INVALID_ARGUMENT || fake::launches) return printf("buffer %d at %d, %ld bytes on\n", result, other, d), 1;
            if (call(result, to + others) || call(result, to - size) || fake::launches != 4) return printf("buffer %d beside %d\n", result, other), 1;
            fake::launches = 0;
        }
    if (call(0, 0) || fake::launches != 2) return printf("buffers apart\n"), 1;
    return 0;
}
""")
    r = run(exe)
    assert r.returncode == 0, r.stdout


def test_the_arrays_struct_is_as_it_was(tmp_path):
    """Programs hand over a struct of eight addresses; the numbers of drafts are had by a call of their own."""
    exe = program(tmp_path, ["kv_dev", "kv"], STUBS + r"""
int main() {
    dc_ctx ctx;
    dc_kv_cache *kv = nullptr, *plain = nullptr;
    if (dc_b200_kv_create_dev(&ctx, 1, 8, 2, 64, DC_GGML_TYPE_BF16, 60, 4, 40, 100, &kv) || dc_b200_kv_create(&ctx, 1, 2, 128, 9, 2, 4, &plain)) return printf("create\n"), 1;
    struct { dc_kv_dev_arrays a; const void* behind; } x = {{}, &ctx};
    const int32_t* drafts = nullptr;
    if (sizeof(x.a) != 8 * sizeof(void*) || dc_b200_kv_dev_arrays(kv, &x.a) || x.behind != &ctx) return printf("the struct\n"), 1;
    if (dc_b200_kv_dev_drafts(kv, &drafts) || !drafts) return printf("drafts\n"), 1;
    for (int s = 0; s < 4; ++s)
        if (drafts[s] != -1 || x.a.counts[s] != 0) return printf("before a step\n"), 1;
    if (dc_b200_kv_dev_drafts(kv, nullptr) != DC_B200_INVALID_ARGUMENT || dc_b200_kv_dev_drafts(nullptr, &drafts) != DC_B200_INVALID_ARGUMENT || dc_b200_kv_dev_drafts(plain, &drafts) != DC_B200_INVALID_ARGUMENT)
        return printf("refusals\n"), 1;
    dc_b200_kv_destroy(kv), dc_b200_kv_destroy(plain);
    return fake::bad_frees || !fake::live.empty();
}
""")
    r = run(exe)
    assert r.returncode == 0, r.stdout
