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
