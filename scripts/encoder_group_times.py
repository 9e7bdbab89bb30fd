"""Times of BasicEncoder(norm_fn='group') on 320 x 512 images, ms: its modules one by
one with NCHW maps, the same in channels last, and the fused norms; fp16 autocast,
fp32, and a module in fp16; forward alone and with gradients.  20 passes after 5.
Result: profiles/operators/encoder_times.txt."""
import copy
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "droid-slam_amd"))
from droid_mi355x.extractor import BasicEncoder  # noqa: E402


def modules_channels_last(enc, x):
    y = x.flatten(0, 1).contiguous(memory_format=torch.channels_last)
    y = enc.relu1(enc.norm1(enc.conv1(y)))
    for layer in (enc.layer1, enc.layer2, enc.layer3):
        for blk in layer:
            y = blk.forward_reference(y)
    return enc.conv2(y)


def ms(enc, run, x, autocast, train):
    def once():
        with torch.set_grad_enabled(train), torch.autocast("cuda", dtype=torch.float16, enabled=autocast):
            y = run(enc, x)
        if train:
            y.float().sum().backward()

    for _ in range(5):
        once()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(20):
        once()
    end.record()
    torch.cuda.synchronize()
    return start.elapsed_time(end) / 20


torch.manual_seed(0)
for frames in (2, 28):
    enc = BasicEncoder(128, "group").cuda()
    x = torch.randn(1, frames, 3, 320, 512, device="cuda")
    for kind in ("fp16 autocast", "fp32", "module in fp16"):
        e, v = (copy.deepcopy(enc).half(), x.half()) if kind == "module in fp16" else (copy.deepcopy(enc), x)
        for train in (False, True):
            times = [ms(e, lambda m, t: m.forward_reference(t), v, kind == "fp16 autocast", train),
                     ms(copy.deepcopy(e).to(memory_format=torch.channels_last), modules_channels_last, v,
                        kind == "fp16 autocast", train),
                     ms(e, lambda m, t: m(t), v, kind == "fp16 autocast", train)]
            print("%2d frames, %-14s %-15s modules NCHW %6.2f  channels last %6.2f  fused %6.2f"
                  % (frames, kind, "with gradients" if train else "forward", *times), flush=True)
