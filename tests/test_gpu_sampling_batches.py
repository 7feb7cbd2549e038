"""Sampled sequences in batches whose heads run in parts: each draws what it draws when it is stepped alone, at temperatures that spread its tokens."""
import pytest

from superslm_b200 import abi, artifact as A

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [40, 257, 300])
@pytest.mark.parametrize("all_sampled", [False, True])
def test_rows_draw_what_they_draw_alone(gpu_lib, rows, all_sampled):
    """other records, scales and numbers than its neighbours' for every row"""
    art = A.build_synthetic_model("tiny", 0xC1, 48)
    eng = abi.Engine(gpu_lib, art, blocks=rows + 1, max_batch=rows, max_chunk=64)
    kinds = (dict(temperature=0.8), dict(temperature=1.3, top_k=40), dict(temperature=1.1, top_p=0.9), dict(temperature=0.9, min_p=0.01), dict(temperature=1.7, top_k=200, top_p=0.95))
    try:
        seqs, prompts, settings = [], [], []
        for i in range(rows):
            s = eng.new_seq()
            p = A.stream_uniform(i, "prompt", 4 + i % 23, 0, 100)
            s.prefill(p, 64)
            c = dict(kinds[i % 5], seed=1000 + i) if all_sampled or i % 3 or i == 256 else None
            if c is not None:
                s.set_sampling(**c)
            seqs.append(s)
            prompts.append(p)
            settings.append(c)
        got = []
        for _ in range(4):
            st, toks = eng.decode_step(seqs, eng.num_layers)
            assert st == 0
            got.append(toks)
        alone, drawn = eng.new_seq(), {False: 0, True: 0}
        for i in range(rows) if rows < 256 else sorted(set(range(0, rows, 7)) | set(range(250, min(rows, 262)))):
            alone.reset()
            alone.set_sampling(temperature=None)
            alone.prefill(prompts[i], 64)
            greedy = alone.decode(4, eng.num_layers)
            if settings[i] is not None:
                alone.reset()
                alone.set_sampling(**settings[i])
                alone.prefill(prompts[i], 64)
                own = alone.decode(4, eng.num_layers)
                drawn[i >= 256] += own != greedy
            else:
                own = greedy
            assert own == [t[i] for t in got], (i, settings[i])
        assert drawn[False] >= 10 and (rows < 300 or drawn[True] >= 4)      # (tokens that hang on the draw, on both sides of a part's end)
    finally:
        eng.close()
