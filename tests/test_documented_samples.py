"""The documented sequence from hidden states to the sampler and the drafter's step compiles against the headers with
every name of the type that its comments give it: a device array that is passed by the address of its pointer does
not."""
import glob
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NAMES = """
#include <cfloat>
#include <cstddef>
#include <cstdint>
#include "ds41_moe_gfx950.h"
#include "ds41_logits_gfx950.h"
#define CK(x) do { const int rc = (x); (void)rc; } while (0)
void sample(void *stream, uint32_t *counts, uint32_t *seen, const uint32_t *grammar, size_t words, int table_rows, int V, int H, int T, int k,
            const int32_t *dev_seq, const int32_t *prompt, const int32_t *prompt_offsets, int prompt_len, const int32_t *drafts,
            const uint16_t *hidden, const uint16_t *head_w, float *target, const float *draft, const float *draft_raw, float *grad,
            const float *penalties, const int32_t *bias_ids, const float *bias_values, const int32_t *bias_offsets, int n_bias,
            int32_t *top_ids, float *top_logits, float *top_lse, const float *grad_loss, float *loss, float *stats, double temp, double top_p,
            unsigned long long seed, unsigned long long step, ds41_spark_result *result, void *ws, void *top_ws, void *accept_ws,
            void *distill_ws, size_t ws_bytes, size_t top_ws_bytes, size_t accept_ws_bytes, size_t distill_ws_bytes) {
%s
}
"""


def test_sequence_around_the_samplers_compiles(tmp_path):
    blocks = [b for f in glob.glob(os.path.join(ROOT, "*.md")) for b in re.findall(r"```cpp\n(.*?)```", open(f).read(), flags=re.S)
              if "ds41_token_counts_add(" in b]
    assert blocks
    for b in blocks:
        src = tmp_path / "sample.cpp"
        src.write_text(NAMES % b)
        r = subprocess.run(["g++", "-std=c++17", "-fsyntax-only", "-Wall", "-Werror", "-I" + os.path.join(ROOT, "include"), str(src)],
                           capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stderr
