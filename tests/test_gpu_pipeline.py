"""StreamPipeline at the size of the bf16 / ViT-base workload: steps queued one behind the other without a synchronisation give the bits of the same steps
one by one, and the two models do not run together."""
import pytest
import torch

from evfly_amd import synthetic as syn
from evfly_amd import vitfly_models as vm

pytestmark = pytest.mark.gpu


def _composite(device):
    import evfly_amd.learner_models as lm
    net = lm.OrigUNet_w_VITFLY_ViTLSTM(vit_trunk=vm.BASE, num_in_channels=2, num_out_channels=1, num_recurrent=[1, 0], input_shape=[1, 1, 260, 346], velpred=0,
                                       form_BEV=2, evs_min_cutoff=0.15, skip_type="interp", logger=lambda *a: None)
    net.load_state_dict(syn.fill_state_dict(net.state_dict()))
    net.set_compute_dtype("bf16")
    return net.to(device).float().eval()


def test_steps_queued_together_equal_steps_one_by_one(gpu_device):
    from evfly_amd.pipeline import StreamPipeline
    S, T = 256, 10
    pipe = StreamPipeline(_composite(gpu_device))
    x = torch.from_numpy(syn.make_frames(41, 64)).cuda().clamp(-1, 1).reshape(64, 1, 260, 346)
    x = (x.repeat(S * T // 64, 1, 1, 1) * torch.linspace(0.6, 1.0, S * T, device="cuda").view(-1, 1, 1, 1)).contiguous()
    desvel = torch.full((S * T, 1), 4.0, device="cuda")
    host = [torch.empty(S * T, 3).pin_memory() for _ in range(4)]
    with torch.no_grad():
        d0, _, _ = pipe.unet.forward_streams(x, None, S, T)
        v0, _ = pipe.vit._run([d0, desvel, None], S, T, clip2x=1)
        torch.cuda.synchronize()
        for rep in range(6):
            outs = [pipe.step(x, desvel, S, T, after=lambda v, i=i: host[i].copy_(v, non_blocking=True)) for i in range(4)]
            torch.cuda.synchronize()
            for i, (v, (d, _, _), _) in enumerate(outs):
                assert torch.equal(d, d0) and torch.equal(v, v0) and torch.equal(host[i], v0.cpu()), (rep, i)
            del outs


def test_a_step_is_ordered_on_the_callers_stream(gpu_device):
    """What a step returns may be read on the stream it was called on, and the velocity model has ended before anything queued behind the step begins."""
    from evfly_amd.pipeline import StreamPipeline
    pipe = StreamPipeline(_composite(gpu_device))
    S, T = 2, 2
    x = torch.from_numpy(syn.make_frames(42, S * T)).cuda().clamp(-1, 1).reshape(S * T, 1, 260, 346)
    desvel = torch.full((S * T, 1), 4.0, device="cuda")
    end = torch.cuda.Event(enable_timing=True)
    begin = torch.cuda.Event(enable_timing=True)

    def after(vel):
        torch.cuda._sleep(20_000_000)                                        # (some milliseconds behind the velocities, on the side stream)
        end.record()
        return vel * 2

    with torch.no_grad():
        pipe.step(x, desvel, S, T)
        vel, _, twice = pipe.step(x, desvel, S, T, after=after)
        begin.record()
        three = vel + twice
    torch.cuda.synchronize()
    assert end.elapsed_time(begin) >= 0
    assert torch.equal(three, vel * 3)
