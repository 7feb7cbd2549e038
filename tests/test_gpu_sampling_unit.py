"""What a logit unit is worth in a decode step, from the model's real numbers: weights of the head and of the final norm are their codes / 127, and the row
that the head multiplies is held in 127ths of its largest element."""
import numpy as np
import pytest

from superslm_b200 import artifact as A
from tests.test_gpu_sampling import engine, step, traced

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", ["tiny", "small", "mini0.5b"])
@pytest.mark.parametrize("temperature", [0.7, 2.0])
def test_draws_are_from_the_softmax_of_real_logits(gpu_lib, shape, temperature):
    """The token is where the distribution function passes its random number. The engine's unit is off by 2^-15 of itself at most (the norm's root by 2^-20, its
    quotients by 2^-16, the scales' products by 2^-29), which moves a weight d octaves down by 2^-15 d ln 2 of itself, and a sum of them by the mean of that,
    twice over in a quotient; the weights' polynomial moves it by 1.4e-5."""
    eng = engine(gpu_lib, shape, 96, 1)
    steps = 40
    numbers = [int(t) for t in np.random.default_rng(5).integers(0, 1 << 31, steps)]
    gain = eng.art.tensors(A.SEC_WEIGHTS, np.int8)["final_norm.gain"].astype(np.float64) / 127
    try:
        s = eng.new_seq()
        traced(eng, lambda: s.prefill(A.stream_uniform(3, "prompt", 9, 0, 100), 64), 8)
        s.set_sampling(temperature=temperature, draws=numbers)
        wrong = {1.0: 0, 0.9: 0, 1.1: 0}
        for n in range(steps):
            toks, rows = step(eng, [s])
            h = np.frombuffer(eng.records[(8 + n, eng.num_layers - 1, 11)][2], dtype=np.int8).astype(np.float64)
            y = h / np.sqrt((h * h).mean()) * gain
            for times in wrong:
                x = rows[0].astype(np.float64) * (np.abs(y).max() / 127 / 127) * times / temperature
                d = x.max() - x
                p = np.exp(-d) / np.exp(-d).sum()
                off = 2 * 2.0 ** -15 * (p * d).sum() + 1.4e-5
                upto, u = np.cumsum(p), numbers[n] / 2.0 ** 31
                wrong[times] += not (upto[toks[0]] >= u - off and upto[toks[0]] - p[toks[0]] <= u + off)
        assert wrong[1.0] == 0 and wrong[0.9] > 0 and wrong[1.1] > 0, wrong
    finally:
        eng.close()
