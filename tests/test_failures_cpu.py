"""Host code around the GPU's: what is left behind, and what still works, once a call of CUDA's runtime has failed."""
from host_util import program, run


def test_a_step_that_outgrows_its_plan_survives_every_failing_call(tmp_path):
    """A cache's plan grows while the n-th call fails, for every n: nothing is freed twice or lost, and the step begins once the call succeeds."""
    exe = program(tmp_path, ["attn_q4", "kv"], r"""
#include "dc_kv.h"
#include "dc_q4.h"
int dc_launch_q4_prompt(dc_ctx*, const dc_q4_call&) { return 0; }
int dc_launch_q4_join(dc_ctx*, const dc_q4_call&) { return 0; }
int main() {
    for (int n = 1;; ++n) {
        dc_ctx ctx;
        dc_kv_cache* kv = nullptr;
        int a = -1, b = -1, st, zero[2] = {0, 0}, few[2] = {3, 1}, many[2] = {4000, 5}, seqs[2], kept[2] = {3, 1};
        fake::fail_at = 0;
        st = dc_b200_kv_create_q4(&ctx, 1, 8, 2, 128, DC_GGML_TYPE_BF16, 600, 2, 400, &kv);
        if (st || dc_b200_kv_seq_alloc(kv, &a) || dc_b200_kv_seq_alloc(kv, &b)) return printf("create: %d\n", st), 1;
        seqs[0] = a, seqs[1] = b;
        if (dc_b200_kv_batch(kv, 2, seqs, zero, few)) return printf("first step\n"), 1;
        fake::calls = 0, fake::fail_at = n;
        st = dc_b200_kv_batch(kv, 2, seqs, kept, many);
        const bool failed = fake::calls >= n;
        fake::fail_at = 0;
        if (failed != (st != 0)) return printf("call %d: status %d\n", n, st), 1;
        if (failed) {
            if (kv->seqs[a].len != 3 || kv->seqs[b].len != 1) return printf("call %d: lengths\n", n), 1;
            if (dc_b200_kv_q4_write_dev(&ctx, kv, 0, &ctx, &ctx, 0, nullptr, nullptr) != DC_B200_INVALID_ARGUMENT) return printf("call %d: the step counts\n", n), 1;
        }
        if ((st = dc_b200_kv_batch(kv, 2, seqs, kept, many))) return printf("call %d, once more: status %d\n", n, st), 1;
        if ((st = dc_b200_kv_q4_write_dev(&ctx, kv, 0, &ctx, &ctx, 0, nullptr, nullptr))) return printf("call %d, rows: status %d\n", n, st), 1;
        dc_b200_kv_destroy(kv);
        if (fake::bad_frees || !fake::live.empty()) return printf("call %d: %d freed twice, %d lost\n", n, fake::bad_frees, (int)fake::live.size()), 1;
        if (!failed) return printf("%d calls\n", n - 1), 0;
    }
}
""")
    r = run(exe)
    assert r.returncode == 0 and int(r.stdout.split()[0]) > 8, r.stdout


def test_sets_of_adapters_beyond_any_memory_are_refused(tmp_path):
    """Sizes whose bytes wrap around 64 bits would get a small allocation and be written far beyond it."""
    exe = program(tmp_path, ["lora"], r"""
extern "C" int dc_b200_mul_mat_dev(dc_ctx*, const dc_weight*, const float*, int, float*) { return 0; }
int main() {
    dc_ctx ctx;
    const long long bad[][4] = {{1 << 24, 1 << 24, 1 << 27, 4096}, {1 << 24, 8, 1 << 27, 4096}, {16, 1 << 24, 1 << 30, 2048}, {1 << 24, 1 << 24, 1 << 28, 16}, {1 << 24, 1 << 24, 2147483647, 4096}, {1 << 23, 100, 1 << 28, 4096}};
    for (auto& b : bad) {
        dc_lora* l = nullptr;
        const int st = dc_b200_lora_create(&ctx, b[0], b[1], (int)b[2], (int)b[3], DC_GGML_TYPE_BF16, &l);
        if (st != DC_B200_OUT_OF_MEMORY || l || fake::calls) return printf("%lld x %lld, %lld adapters of rank %lld: status %d\n", b[0], b[1], b[2], b[3], st), 1;
    }
    dc_lora* l = nullptr;
    if (dc_b200_lora_create(&ctx, 64, 32, 4, 8, DC_GGML_TYPE_BF16, &l)) return printf("a small one\n"), 1;
    dc_b200_lora_destroy(l);
    return fake::bad_frees || !fake::live.empty();
}
""")
    r = run(exe)
    assert r.returncode == 0, r.stdout


def test_a_set_of_adapters_that_fails_to_be_made_leaves_nothing(tmp_path):
    exe = program(tmp_path, ["lora"], r"""
extern "C" int dc_b200_mul_mat_dev(dc_ctx*, const dc_weight*, const float*, int, float*) { return 0; }
int main() {
    for (int n = 1;; ++n) {
        dc_ctx ctx;
        dc_lora* l = nullptr;
        fake::calls = 0, fake::fail_at = n;
        const int st = dc_b200_lora_create(&ctx, 64, 32, 4, 8, DC_GGML_TYPE_BF16, &l);
        const bool failed = fake::calls >= n;
        if (failed != (st != 0) || failed != !l) return printf("call %d: status %d\n", n, st), 1;
        dc_b200_lora_destroy(l);
        if (fake::bad_frees || !fake::live.empty()) return printf("call %d: %d freed twice, %d lost\n", n, fake::bad_frees, (int)fake::live.size()), 1;
        if (!failed) return printf("%d calls\n", n - 1), 0;
    }
}
""")
    r = run(exe)
    assert r.returncode == 0 and int(r.stdout.split()[0]) == 6, r.stdout


def test_a_product_with_adapters_is_refused_before_any_of_it_runs(tmp_path):
    """Too many rows, or a workspace that cannot grow (a capture, no memory): neither the product nor anything else has been enqueued."""
    exe = program(tmp_path, ["lora"], r"""
static int products = 0;
extern "C" int dc_b200_mul_mat_dev(dc_ctx*, const dc_weight*, const float*, int, float*) { return ++products, 0; }
int main() {
    dc_ctx ctx;
    dc_weight w = {};
    w.K = 256, w.N = 32, w.E = 1;
    dc_lora* l = nullptr;
    if (dc_b200_lora_create(&ctx, 256, 32, 4, 8, DC_GGML_TYPE_BF16, &l)) return printf("create\n"), 1;
    float* x = (float*)(size_t(1) << 40);      // (nothing reads them here)
    float* y = (float*)(size_t(1) << 44);
    const int* ids = (const int*)x;
    auto refused = [&](int M, int status) {
        fake::launches = products = 0;
        const int st = dc_b200_mul_mat_lora_dev(&ctx, &w, l, x, M, ids, y);
        if (st != status || products || fake::launches) printf("%d rows: status %d, %d products\n", M, st, products), exit(1);
    };
    refused(65535 * 16 + 1, DC_B200_INVALID_ARGUMENT);
    fake::capturing = true;
    refused(5, DC_B200_UNSUPPORTED);
    fake::capturing = false;
    fake::calls = 0, fake::fail_at = 1;
    refused(5, DC_B200_OUT_OF_MEMORY);
    fake::fail_at = 0;
    if (dc_b200_mul_mat_lora_dev(&ctx, &w, l, x, 5, ids, y) || products != 1 || fake::launches != 2) return printf("five rows: %d products, %d launches\n", products, fake::launches), 1;
    fake::capturing = true;
    if (dc_b200_mul_mat_lora_dev(&ctx, &w, l, x, 5, ids, y) || products != 2) return printf("five rows, captured\n"), 1;
    refused(4000, DC_B200_UNSUPPORTED);
    dc_b200_lora_destroy(l);
    return fake::bad_frees || !fake::live.empty();
}
""")
    r = run(exe)
    assert r.returncode == 0, r.stdout


def test_a_cache_that_fails_to_be_made_leaves_nothing(tmp_path):
    exe = program(tmp_path, ["attn_q4", "kv"], r"""
#include "dc_kv.h"
#include "dc_q4.h"
int dc_launch_q4_prompt(dc_ctx*, const dc_q4_call&) { return 0; }
int dc_launch_q4_join(dc_ctx*, const dc_q4_call&) { return 0; }
int main() {
    for (int n = 1;; ++n) {
        dc_ctx ctx;
        dc_kv_cache* kv = nullptr;
        fake::calls = 0, fake::fail_at = n;
        const int st = dc_b200_kv_create_q4(&ctx, 3, 8, 2, 64, DC_GGML_TYPE_F32, 60, 2, 40, &kv);
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
