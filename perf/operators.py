"""Cases of the encoder-training operators: group norm with its activation and
residual add (channels last), and the two losses over the all-pairs correlation
of feature maps - softmax cross entropy against a correspondence, and
distillation from a teacher's top logits.

`run` computes an operator in elementary torch operations where `own` is false,
and through the framework's entry points where it is true.  Sizes follow the
320x512 images (maps of 160x256, 80x128 and 40x64) and the training clips of 7
frames and 24 edges the encoders are used with, and generic odd ones."""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
SCALE = 1.0 / 16.0      # CorrBlock's logits: both feature maps over 4
EPS = 1e-5
MODES = ("relu", "res_relu", "add_relu", "none", "silu")   # the entry points' mode numbers, in order


def _gn(name, train, dtype, n, c, groups, h, w, mode):
    return {"name": name, "op": "gn", "train": train, "dtype": dtype, "n": n, "c": c, "groups": groups,
            "h": h, "w": w, "mode": mode}


def _corr(name, op, train, dtype, clips, frames, edges, h, w, dim, points=0, topk=0):
    return {"name": name, "op": op, "train": train, "dtype": dtype, "clips": clips, "frames": frames, "edges": edges,
            "h": h, "w": w, "dim": dim, "points": points, "topk": topk}


def listed():
    return [
        # one frame's 1/8 map while tracking: the smallest call, launch latency
        _gn("gn_frame_eighth", False, "fp16", 1, 128, 16, 40, 64, "relu"),
        # a stereo frame's first norm (8 groups of 4 channels) at half resolution
        _gn("gn_stereo_half", False, "fp16", 2, 32, 8, 160, 256, "relu"),
        # four training clips of 7 frames: a residual block's last norm at half resolution, under bf16 autocast
        _gn("gn_train_half", True, "bf16", 28, 32, 4, 160, 256, "res_relu"),
        # the strided block's shortcut norm at quarter resolution, training in fp32
        _gn("gn_train_quarter", True, "fp32", 28, 64, 8, 80, 128, "add_relu"),
        # odd map and channel counts, smooth activation
        _gn("gn_train_odd", True, "fp16", 3, 60, 12, 61, 83, "silu"),
        # validation of one frame pair, both directions: few rows
        _corr("xent_val_pair", "xent", False, "fp16", 1, 2, 2, 30, 40, 128),
        # one training clip: 7 frames, 24 edges
        _corr("xent_train_clip", "xent", True, "fp16", 1, 7, 24, 40, 64, 128),
        # a batch of four clips: the largest
        _corr("xent_train_batch", "xent", True, "bf16", 4, 7, 24, 40, 64, 128),
        # sampled query points against whole quarter-resolution maps: the longest vocabulary
        _corr("xent_train_points", "xent", True, "bf16", 1, 6, 30, 80, 128, 128, points=501),
        # sub-pixel correspondences: the four bilinear neighbours as soft targets
        _corr("distill_train_subpixel", "distill", True, "fp16", 1, 7, 24, 40, 64, 128, topk=4),
        # a teacher's 16 best matches a pixel, batch of four clips
        _corr("distill_train_top16", "distill", True, "bf16", 4, 7, 24, 40, 64, 128, topk=16),
        # validation of a narrow student on odd maps
        _corr("distill_val_odd", "distill", False, "fp16", 1, 3, 5, 37, 53, 72, topk=7),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _unnamed(case):
    return {k: v for k, v in case.items() if k != "name"}


def draw(rng):
    top_gn = 28 * 32 * 160 * 256
    top_corr = 96 * 2560 * 2560 * 128
    if rng.random() < 0.4:
        while True:
            groups = _log(rng, 1, 32)
            c = groups * _log(rng, 1, 16)
            n, h, w = _log(rng, 1, 28), _log(rng, 5, 160), _log(rng, 5, 256)
            if c <= 256 and 2000 <= n * c * h * w <= top_gn:
                break
        return _unnamed(_gn(None, rng.random() < 0.6, rng.choice(["fp16", "bf16", "fp32"]), n, c, groups, h, w,
                            rng.choice(MODES)))
    op = rng.choice(["xent", "distill"])
    while True:
        clips, frames = rng.choice([1, 1, 2, 3, 4]), rng.randint(2, 9)
        edges = rng.randint(1, min(24, frames * (frames - 1)))
        h, w = _log(rng, 8, 80), _log(rng, 8, 128)
        dim = rng.choice([32, 64, 72, 96, 128, 128, 128])
        points = _log(rng, 100, 1000) if rng.random() < 0.25 else 0
        rows = clips * edges * (points or h * w)
        topk = rng.choice([1, 2, 4, 4, 7, 8, 16]) if op == "distill" else 0
        if rows * h * w * 128 <= top_corr and topk < h * w:
            break
    return _unnamed(_corr(None, op, rng.random() < 0.6, rng.choice(["fp16", "bf16"]), clips, frames, edges, h, w, dim,
                          points, topk))


# ---- inputs ---------------------------------------------------------------

def _edges(case):
    """The nearest ordered pairs of each clip's frames, as a training graph has them."""
    F, E = case["frames"], case["edges"]
    pairs = sorted(((abs(i - j), i, j) for i in range(F) for j in range(F) if i != j))[:E]
    ii = [k * F + i for k in range(case["clips"]) for _, i, _ in pairs]
    jj = [k * F + j for k in range(case["clips"]) for _, _, j in pairs]
    return ii, jj


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DT[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    if case["op"] == "gn":
        n, c, h, w = case["n"], case["c"], case["h"], case["w"]

        def act(t):     # (n, c, h, w) in channels_last memory
            return t.to(dt).permute(0, 3, 1, 2)

        # a convolution's output: channels with their own scale and offset
        x = act(randn(n, h, w, c) * (0.5 + torch.rand(c, generator=g, device=DEV)) + 0.3 * randn(c))
        s = {"case": case, "x": x, "w": 1 + 0.1 * randn(c), "b": 0.1 * randn(c), "res": None}
        if case["mode"] in ("res_relu", "add_relu"):
            s["res"] = act(randn(n, h, w, c).clamp_(min=0))     # the block's input: after a ReLU
        if case["train"]:
            s["dy"] = act(randn(n, h, w, c))
            for k in ("x", "w", "b", "res"):
                if s[k] is not None:
                    s[k].requires_grad_(True)
        return s

    h, w, dim, P = case["h"], case["w"], case["dim"], case["points"]
    Q, N = h * w, case["clips"] * case["frames"]
    # every frame sees the same scene shifted by a few pixels a frame, with noise of its own
    ii, jj = _edges(case)
    scene = randn(case["clips"], h, w, dim)
    sy = torch.randint(-2, 3, (N,), generator=g, device=DEV)
    sx = torch.randint(-3, 4, (N,), generator=g, device=DEV)
    ys, xs = torch.arange(h, device=DEV), torch.arange(w, device=DEV)
    clip = torch.arange(N, device=DEV) // case["frames"]
    at_y = (ys[None, :, None] + sy[:, None, None]) % h
    at_x = (xs[None, None, :] + sx[:, None, None]) % w
    fmaps = (0.9 * scene[clip[:, None, None], at_y, at_x] + 0.45 * randn(N, h, w, dim)).to(dt)
    ii_d = torch.tensor(ii, dtype=torch.int32, device=DEV)
    jj_d = torch.tensor(jj, dtype=torch.int32, device=DEV)
    il, jl = ii_d.long(), jj_d.long()
    # pixel p of frame i is at p + shift_i - shift_j in frame j; outside the map: no correspondence
    ty = ys[None, :, None] + (sy[il] - sy[jl])[:, None, None]
    tx = xs[None, None, :] + (sx[il] - sx[jl])[:, None, None]
    seen = (ty >= 0) & (ty < h) & (tx >= 0) & (tx < w)
    target = torch.where(seen, ty * w + tx, -1).reshape(len(ii), Q)
    s = {"case": case, "f1": ii_d, "f2": jj_d, "fmap1": fmaps.reshape(N, Q, dim), "fmap2": None}
    if P:
        at = torch.randint(0, Q, (N, P), generator=g, device=DEV)
        s["fmap2"] = s["fmap1"]
        s["fmap1"] = torch.gather(s["fmap2"], 1, at[:, :, None].expand(N, P, dim)).contiguous()
        target = torch.gather(target, 1, at[il])
    R = target.shape[1]
    if case["op"] == "xent":
        s["target"] = target.to(torch.int32).contiguous()
    else:
        K = case["topk"]
        # the teacher's best matches: distinct pixels around the correspondence, the nearer the stronger
        off = sorted(((dy * dy + dx * dx, dy * w + dx) for dy in range(-5, 6) for dx in range(-5, 6)))
        seen_off, offs = set(), []
        for d2, o in off:
            if o % Q not in seen_off and len(offs) < K:
                seen_off.add(o % Q)
                offs.append((d2, o))
        while len(offs) < K:
            o = len(offs) + 6 * w
            offs.append((50, o))
        o = torch.tensor([o for _, o in offs], device=DEV)
        d2 = torch.tensor([float(d) for d, _ in offs], device=DEV)
        idx = (target[:, :, None] + o) % Q
        idx = torch.where((target >= 0)[:, :, None], idx, torch.full_like(idx, -1))
        s["idx"] = idx.to(torch.int32).contiguous()
        s["logits"] = (9.0 - 0.8 * d2 + 0.7 * randn(len(ii), R, K)).contiguous()
        s["temp"] = 2.0 if K > 4 else 1.0
    if case["train"]:
        # a mean over the pixels, weighted by a confidence; with fp16 features under a gradient scaler
        loss_scale = 65536.0 if case["dtype"] == "fp16" else 1.0
        s["g"] = torch.rand((len(ii), R), generator=g, device=DEV) * (loss_scale / (len(ii) * R))
        for k in ("fmap1", "fmap2"):
            if s[k] is not None:
                s[k].requires_grad_(True)
    return s


# ---- the plain forms ------------------------------------------------------

def _plain_gn(s):
    case = s["case"]
    n, c, h, w, G = case["n"], case["c"], case["h"], case["w"], case["groups"]
    mode, train = case["mode"], case["train"]

    def rows(t):
        return t.detach().permute(0, 2, 3, 1).reshape(n, h, w, G, c // G)

    def back(t):
        return t.reshape(n, h, w, c).to(DT[case["dtype"]]).permute(0, 3, 1, 2)

    wt, b = s["w"].detach().view(G, c // G), s["b"].detach().view(G, c // G)
    x = rows(s["x"]).float()
    res = None if s["res"] is None else rows(s["res"]).float()
    if train:
        # where a ReLU cuts, the sign of a value next to zero decides a whole gradient: that comparison in 64 bits
        xd = x.double()
        md = xd.mean((1, 2, 4), keepdim=True)
        rd = ((xd - md).square().mean((1, 2, 4), keepdim=True) + EPS).rsqrt()
        mean, rstd = md.float(), rd.float()
        nd = (xd - md) * rd * wt.double() + b.double()
    else:
        mean = x.mean((1, 2, 4), keepdim=True)
        rstd = ((x - mean).square().mean((1, 2, 4), keepdim=True) + EPS).rsqrt()
    xhat = (x - mean) * rstd
    y = xhat * wt + b
    if mode == "relu":
        y = y.clamp(min=0)
    elif mode == "res_relu":
        y = (res + y.clamp(min=0)).clamp(min=0)
    elif mode == "add_relu":
        y = (y + res).clamp(min=0)
    elif mode == "silu":
        z = y
        y = z / (1 + torch.exp(-z))
    if not train:
        return back(y)
    dy = rows(s["dy"]).float()
    dres = None
    if mode == "relu":
        dn = dy * (nd > 0)
    elif mode == "res_relu":
        dres = dy * (res.double() + nd.clamp(min=0) > 0)
        dn = dres * (nd > 0)
    elif mode == "add_relu":
        dres = dy * (nd + res.double() > 0)
        dn = dres
    elif mode == "silu":
        sg = 1 / (1 + torch.exp(-z))
        dn = dy * sg * (1 + z * (1 - sg))
    else:
        dn = dy
    dw = (dn * xhat).sum((0, 1, 2)).reshape(c)
    db = dn.sum((0, 1, 2)).reshape(c)
    dxh = dn * wt
    dx = rstd * (dxh - dxh.mean((1, 2, 4), keepdim=True) - xhat * (dxh * xhat).mean((1, 2, 4), keepdim=True))
    out = {"y": back(y), "dx": back(dx), "dw": dw, "db": db}
    if dres is not None:
        out["dres"] = back(dres)
    return out


def _plain_corr(s):
    case = s["case"]
    fmap1 = s["fmap1"].detach()
    fmap2 = fmap1 if s["fmap2"] is None else s["fmap2"].detach()
    i, j = s["f1"].long(), s["f2"].long()
    a, b = fmap1[i].float(), fmap2[j].float()                       # (E, P, D), (E, Q, D)
    T = s.get("temp", 1.0)
    logits = torch.bmm(a, b.transpose(1, 2).contiguous()) * (SCALE / T)
    top = logits.max(2, keepdim=True).values
    p = torch.exp(logits - top)
    total = p.sum(2, keepdim=True)
    lse = (top + torch.log(total)).squeeze(2)
    if case["op"] == "xent":
        idx = s["target"].long()[:, :, None]
        pi = torch.ones_like(idx, dtype=torch.float32)
        neg_entropy = 0.0
    else:
        idx = s["idx"].long()
        t = (s["logits"] / T).masked_fill(idx < 0, -math.inf)
        t = t - t.max(2, keepdim=True).values
        e = torch.exp(t)
        pi = e / e.sum(2, keepdim=True)
        neg_entropy = torch.where(pi > 0, pi * torch.log(pi), torch.zeros_like(pi)).sum(2)
    used = (idx >= 0).any(2)
    pi = torch.where(idx >= 0, pi, torch.zeros_like(pi))
    at = idx.clamp(min=0)
    loss = neg_entropy + lse - (pi * torch.gather(logits, 2, at)).sum(2)
    loss = torch.where(used, loss, torch.zeros_like(loss)) * (T * T)
    if not case["train"]:
        return loss
    ds = (p / total).scatter_add(2, at, -pi)
    ds = ds * (s["g"] * used * T * SCALE)[:, :, None]
    da, db = torch.bmm(ds, b), torch.bmm(ds.transpose(1, 2).contiguous(), a)
    d1 = torch.zeros_like(fmap1, dtype=torch.float32).index_add_(0, i, da)
    if s["fmap2"] is None:
        return {"loss": loss, "d1": d1.index_add_(0, j, db).to(fmap1.dtype)}
    d2 = torch.zeros_like(fmap2, dtype=torch.float32).index_add_(0, j, db)
    return {"loss": loss, "d1": d1.to(fmap1.dtype), "d2": d2.to(fmap2.dtype)}


# ---- the framework's calls ------------------------------------------------

def _package():
    path = os.path.join(os.getcwd(), "droid-slam_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import droid_backends
    import droid_mi355x
    return droid_backends, droid_mi355x


def _own_gn(s):
    nb, dm = _package()
    case = s["case"]
    mode = MODES.index(case["mode"])
    if not case["train"]:
        return nb.group_norm_act(s["x"], case["groups"], s["w"], s["b"], mode, res=s["res"], eps=EPS)
    y = dm.group_norm_act(s["x"], case["groups"], s["w"], s["b"], mode, res=s["res"], eps=EPS)
    leaves = [s["x"], s["w"], s["b"]] + ([] if s["res"] is None else [s["res"]])
    grads = torch.autograd.grad(y, leaves, s["dy"])
    out = {"y": y.detach(), "dx": grads[0], "dw": grads[1], "db": grads[2]}
    if s["res"] is not None:
        out["dres"] = grads[3]
    return out


def _own_corr(s):
    _, dm = _package()
    case = s["case"]
    if case["op"] == "xent":
        loss = dm.corr_cross_entropy(s["fmap1"], s["fmap2"], s["f1"], s["f2"], s["target"], scale=SCALE)
    else:
        loss = dm.corr_distillation(s["fmap1"], s["fmap2"], s["f1"], s["f2"], s["idx"], s["logits"], scale=SCALE,
                                    temperature=s["temp"])
    if not case["train"]:
        return loss
    if s["fmap2"] is None:
        return {"loss": loss.detach(), "d1": torch.autograd.grad(loss, s["fmap1"], s["g"])[0]}
    d1, d2 = torch.autograd.grad(loss, [s["fmap1"], s["fmap2"]], s["g"])
    return {"loss": loss.detach(), "d1": d1, "d2": d2}


def run(s):
    if own:
        return _own_gn(s) if s["case"]["op"] == "gn" else _own_corr(s)
    return _plain_gn(s) if s["case"]["op"] == "gn" else _plain_corr(s)


# ---- what a pass cannot do without ----------------------------------------

def work(case):
    es = BYTES[case["dtype"]]
    if case["op"] == "gn":
        m = case["n"] * case["c"] * case["h"] * case["w"]
        res = case["mode"] in ("res_relu", "add_relu")
        maps = 2 + res + (2 + res if case["train"] else 0)      # x, y, res; dy, dx, dres
        return {"bytes": maps * m * es + 8 * case["c"] * (2 if case["train"] else 1),
                "flops": m * (30 if case["train"] else 10)}
    Q, E, D = case["h"] * case["w"], case["clips"] * case["edges"], case["dim"]
    P, N, K = case["points"] or Q, case["clips"] * case["frames"], max(1, case["topk"])
    feats = N * Q * D * es + (N * P * D * es if case["points"] else 0)
    rows = E * P * 4 * (1 + (2 * K if case["topk"] else 1))     # the loss, and the targets or the indices and logits
    if not case["train"]:
        return {"bytes": feats + rows, "flops": 2 * E * P * Q * D}
    return {"bytes": 2 * feats + rows + E * P * 4, "flops": 6 * E * P * Q * D}


# ---- the definition, in 64 bits -------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_gn(case, s) if case["op"] == "gn" else _exact_corr(case, s)


def _exact_gn(case, s):
    G, mode = case["groups"], case["mode"]
    w, b = s["w"].double(), s["b"].double()
    y, dx, dres = [], [], []
    dw, db = torch.zeros_like(w), torch.zeros_like(b)
    for k in range(case["n"]):                                   # image by image
        x = s["x"][k].double()                                   # (c, h, w)
        v = x.reshape(G, -1)
        var, mu = torch.var_mean(v, 1, correction=0, keepdim=True)
        inv = 1.0 / torch.sqrt(var + EPS)
        xh = ((v - mu) * inv).reshape(x.shape)
        z = xh * w[:, None, None] + b[:, None, None]
        r = None if s["res"] is None else s["res"][k].double()
        if mode == "relu":
            o, slope, slope_r = torch.relu(z), (z > 0).double(), None
        elif mode == "res_relu":
            o = torch.relu(r + torch.relu(z))
            slope_r = (o > 0).double()
            slope = slope_r * (z > 0)
        elif mode == "add_relu":
            o = torch.relu(z + r)
            slope = slope_r = (o > 0).double()
        elif mode == "silu":
            sg = torch.sigmoid(z)
            o, slope, slope_r = z * sg, sg + z * sg * (1 - sg), None
        else:
            o, slope, slope_r = z, torch.ones_like(z), None
        y.append(o)
        if case["train"]:
            gy = s["dy"][k].double()
            gn = gy * slope
            if slope_r is not None:
                dres.append(gy * slope_r)
            dw += (gn * xh).sum((1, 2))
            db += gn.sum((1, 2))
            gh = (gn * w[:, None, None]).reshape(G, -1)
            xv = xh.reshape(G, -1)
            m = gh.shape[1]
            dx.append((inv * (gh - gh.sum(1, keepdim=True) / m - xv * (gh * xv).sum(1, keepdim=True) / m))
                      .reshape(x.shape))
    if not case["train"]:
        return torch.stack(y)
    out = {"y": torch.stack(y), "dx": torch.stack(dx), "dw": dw, "db": db}
    if dres:
        out["dres"] = torch.stack(dres)
    return out


def _exact_corr(case, s):
    f1 = s["fmap1"].double()
    f2 = f1 if s["fmap2"] is None else s["fmap2"].double()
    d1 = torch.zeros_like(f1)
    d2 = d1 if s["fmap2"] is None else torch.zeros_like(f2)
    T = s.get("temp", 1.0)
    losses = []
    for e, (i, j) in enumerate(zip(s["f1"].tolist(), s["f2"].tolist())):   # edge by edge
        z = (f1[i] @ f2[j].T) * (SCALE / T)
        logp = torch.log_softmax(z, 1)
        q = torch.zeros_like(z)                                  # the targets' distribution, dense
        if case["op"] == "xent":
            t = s["target"][e].long()
            on = t >= 0
            q[on.nonzero()[:, 0], t[on]] = 1.0
        else:
            t = s["idx"][e].long()
            on = (t >= 0).any(1)
            pi = torch.softmax((s["logits"][e].double() / T)[on].masked_fill(t[on] < 0, -math.inf), 1)
            q[on] = q[on].scatter_add(1, t[on].clamp(min=0), pi)
        kl = (torch.xlogy(q, q) - q * logp).sum(1)
        losses.append(torch.where(on, kl, torch.zeros_like(kl)) * (T * T))
        if case["train"]:
            dz = (torch.exp(logp) - q) * (s["g"][e].double() * on * T * SCALE)[:, None]
            d1[i] += dz @ f2[j]
            d2[j] += dz.T @ f1[i]
    loss = torch.stack(losses)
    if not case["train"]:
        return loss
    return {"loss": loss, "d1": d1} if s["fmap2"] is None else {"loss": loss, "d1": d1, "d2": d2}
