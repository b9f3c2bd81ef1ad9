"""A stream of batches through the composite D(theta) -> V(phi) (learner/learner_models.py:618-636), the velocity model on a stream of its own.

`OrigUNet_w_VITFLY_ViTLSTM.forward` is one call per batch, as in the reference. For a STREAM of batches (evfly_ros/run.py:245-268 called at 15 Hz per
camera; bench.py's steps) `StreamPipeline` queues the two models separately, their states kept apart (the ConvLSTM state goes D -> D, the nn.LSTM state
P -> P): D on the caller's stream, P and what follows it (the all_gather, the copy to pinned host memory) on a second HIP stream behind D's event, and the
caller's stream behind P's. Same kernels, same order, same bits as the composite call (tests/test_gpu_models.py::test_stream_pipeline_equals_composite).

The two models do not share the device. Nothing of D(i + 1) needs P(i), but run together they have not been sound: with the bf16 U-Net of 2560 frames and
the ViT-base trunk, 2 to 5 % of the steps whose depth model ran beside a velocity model had wrong depth in the first frames of their second chunk, the
same steps one after the other never. The cause was not found in the kernels; the overlap was worth 1 to 2 %.

No reference counterpart beyond the call pattern above: the reference is single-stream PyTorch.
"""
import torch

from . import _lib


class StreamPipeline:
    def __init__(self, model):
        """model: an `OrigUNet_w_VITFLY_ViTLSTM` on the GPU (its two sub-modules build their own native handles)."""
        _lib.lib()
        self.unet, self.vit = model.origunet, model.vitfly_vitlstm
        name = {0: "f32", 1: "bf16", 2: "bf16x3"}[model.compute_dtype]
        self.unet.set_compute_dtype(name)           # (the setter also thaws a frozen handle: a plain attribute write does not)
        self.vit.set_compute_dtype(name)
        self.side = torch.cuda.Stream()

    def step(self, frames, desvel, n_streams, T, unet_state=None, vit_state=None, after=None):
        """One batch, laid out [stream][t] like `forward_streams`. D runs on the current stream, P on the side stream behind it, then `after(vel)` (e.g. the
        all_gather + copy to pinned host memory), still on the side stream; the current stream goes on behind them. Returns
        (vel, (depth, upconv, ((h_unet, None), (lstm_h, lstm_c))), after's result), all valid on the current stream."""
        main = torch.cuda.current_stream()
        main.wait_stream(self.side)                        # (a step before this one may have been another stream's)
        depth, upconv, h_unet = self.unet.forward_streams(frames, unet_state, n_streams, T)
        self.side.wait_stream(main)
        try:
            with torch.cuda.stream(self.side):
                depth.record_stream(self.side)             # the caching allocator must not recycle it under P
                X = [depth, desvel, None] + ([vit_state] if vit_state is not None else [])
                vel, st = self.vit._run(X, n_streams, T, clip2x=1)  # x_depth_input = clip(2 * depth, 0, 1), learner_models.py:634
                extra = after(vel) if after is not None else None
        finally:
            main.wait_stream(self.side)                    # (also where `after` raises: P is under way by then)
        # vel, the LSTM state and after's result come from the SIDE stream's pool of the caching allocator: their readers are on this stream
        for t in _flatten((vel, st, extra)):
            if isinstance(t, torch.Tensor) and t.is_cuda:
                t.record_stream(main)
        return vel, (depth, upconv, ((h_unet, None), st)), extra

    def wait(self):
        """The results of `step` are ordered on the stream that it was called on; a reader on another stream waits for that one."""
        torch.cuda.current_stream().wait_stream(self.side)


def _flatten(x):
    if isinstance(x, (tuple, list)):
        for y in x:
            yield from _flatten(y)
    else:
        yield x
