"""The gate vectors of a step whose time is met for the first time reach both branches' streams."""
import pytest
import torch

from vdit.runtime import FlowMatchSamplingParams

from tests.test_gpu_forward import build

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("share", [True, False])
def test_first_sample_of_a_schedule_is_the_second_one(share):
    """A schedule other than the runner's own has gates that nothing has computed yet.  They are made late here
    (a delay before them, on the stream that makes them), on memory full of NaN."""
    _, _, runner, vox, ctx, xt = build(512, 128, depth=3, cdepth=2, n=700, side=8, patch=256, seed=31)
    runner.solver_config.ditfastattn_b0_msa_share = share
    vox, ctx, xt = torch.from_numpy(vox).to(DEV), ctx.to(DEV, torch.bfloat16), xt.to(DEV)
    sampling = FlowMatchSamplingParams(guidance_scale=3.0, num_inference_steps=3, rescale_t=2.0)
    known, make = set(runner._time_gates_cache), runner._get_time_gates

    def late(t, *a, **kw):
        if round(float(t), 7) not in runner._time_gates_cache:
            torch.cuda._sleep(100_000_000)                   # about 50 ms
        return make(t, *a, **kw)

    runner.sample_with_context(vox, ctx, noise=xt)           # every kernel set up
    torch.cuda.synchronize()
    full = [torch.full((n,), float("nan"), device=DEV) for n in (1000, 20000, 60000) for _ in range(40)]
    del full
    runner._get_time_gates = late
    first = runner.sample_with_context(vox, ctx, sampling=sampling, noise=xt)
    torch.cuda.synchronize()
    assert set(runner._time_gates_cache) - known             # the schedule did bring new times
    second = runner.sample_with_context(vox, ctx, sampling=sampling, noise=xt)
    assert torch.isfinite(first).all() and torch.equal(first, second)
