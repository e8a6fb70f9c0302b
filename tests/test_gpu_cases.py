"""The timed cases of the 8-bit products and the norm's gates as a program would run them: inputs
just made behind a busy stream, outputs used at once, inputs dropped."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "more_operators.py")


@pytest.mark.parametrize("other", [False, True])
def test_calls_are_ordered_with_their_inputs_and_outputs(other):
    """On the program's own stream, and on one that the caller makes current."""
    import torch
    spec = importlib.util.spec_from_file_location("more_operators", PATH)
    cases = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(cases)
    big = torch.empty(1 << 29, dtype=torch.uint8, device="cuda")
    with torch.cuda.stream(torch.cuda.current_stream()):  # the stream before is current again behind this
        for i, case in enumerate(cases.listed()):
            with torch.cuda.stream(torch.cuda.Stream() if other else torch.cuda.current_stream()):
                cases.own = True
                for k in range(6):
                    big.fill_(k)
                state = cases.prepare(case, i)
                out = cases.run(state)
                got = [o.clone() for o in (out if isinstance(out, tuple) else (out,))]
                del state, out
                cases.own = False
                want = cases.run(cases.prepare(case, i))
                torch.cuda.synchronize()
                want = want if isinstance(want, tuple) else (want,)
                assert all(torch.equal(a, b) for a, b in zip(got, want)), case
        torch.cuda.synchronize()
        for bw in (32, 64):
            cases._ctx[bw].close()
