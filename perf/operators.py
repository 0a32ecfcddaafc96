"""The layer operators of card_amd (dropout, root-mean-square norm, products with 4-bit weights): their cases, their plain
form and their 64-bit values.

A hidden layer of a guidance network or of a conditional head on language-model features is: add the residual, norm, a
product with few rows against 4-bit weights, an activation, dropout.  `run` makes one pass through one of these
operators; where the module's `own` is false it computes the same from elementary torch operations in 32 bits.
"""
import torch

own = False

_DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2, "e4m3": 1}
_M32 = 0xFFFFFFFF
_E4M3_MAX = 448.0


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # Monte-Carlo dropout of a hidden layer of the regression guidance network: 64 test rows, width 100, 100 masks each
        {"name": "drop_mc_rows", "op": "dropout", "dtype": "fp32", "rows": 64, "cols": 100, "n_z": 100, "p": 0.2,
         "residual": False, "train": False},
        # a training step's dropout on the branch of a residual layer, forward and backward
        {"name": "drop_train_bf16", "op": "dropout", "dtype": "bf16", "rows": 8192, "cols": 4096, "n_z": 1, "p": 0.1,
         "residual": True, "train": True},
        # the same at an odd width, three masks a row, an element offset that is no multiple of four
        {"name": "drop_train_odd_fp16", "op": "dropout", "dtype": "fp16", "rows": 1237, "cols": 1501, "n_z": 3, "p": 0.5,
         "residual": False, "train": True},
        # the largest batch: a GiB of fp32 read and written
        {"name": "drop_large_fp32", "op": "dropout", "dtype": "fp32", "rows": 16384, "cols": 8192, "n_z": 1, "p": 0.1,
         "residual": False, "train": False},
        # one token of a 4096-wide layer on its way into a product: residual, norm, 8 bits
        {"name": "norm_token_e4m3", "op": "norm_e4m3", "dtype": "bf16", "rows": 1, "cols": 4096, "residual": True},
        # a batch of prompts
        {"name": "norm_prompt_e4m3", "op": "norm_e4m3", "dtype": "bf16", "rows": 8192, "cols": 4096, "residual": True},
        # a training step at the widest head, forward and backward
        {"name": "norm_train_bf16", "op": "norm", "dtype": "bf16", "rows": 8192, "cols": 6144, "residual": True, "train": True},
        # odd width, fp32, no residual
        {"name": "norm_train_odd_fp32", "op": "norm", "dtype": "fp32", "rows": 1777, "cols": 5003, "residual": False,
         "train": True},
        # a single token through a square 4096 layer (the classification head's width)
        {"name": "w4_token", "op": "w4", "dtype": "bf16", "rows": 1, "in": 4096, "out": 4096, "group": 128, "zero": False,
         "gamma": False},
        # sixteen tokens in 8 bits through a large layer, weights with zero points
        {"name": "w4_tokens_large", "op": "w4", "dtype": "e4m3", "rows": 16, "in": 8192, "out": 28672, "group": 128,
         "zero": True, "gamma": False},
        # a conditional layer in fp32 at odd sizes, small groups: gamma[t] * (W x + b), LeakyReLU
        {"name": "w4_cond_odd_fp32", "op": "w4", "dtype": "fp32", "rows": 5, "in": 1001, "out": 777, "group": 32,
         "zero": True, "gamma": True},
        # norm and product in one go, as a layer of a served network runs them: 24 rows
        {"name": "norm_w4_rows", "op": "norm_w4", "dtype": "bf16", "rows": 24, "in": 4096, "out": 6144, "group": 64,
         "zero": False, "gamma": False},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(("dropout", "norm_e4m3", "norm", "w4", "w4", "norm_w4"))
    dtype = rng.choice(("fp32", "bf16", "fp16"))
    if op == "dropout":
        cols, n_z = _log(rng, 1, 16384), rng.choice((1, 1, 1, rng.randint(2, 64)))
        rows = _log(rng, 1, max(1, min(100_000, 40_000_000 // (cols * n_z))))
        return {"op": op, "dtype": dtype, "rows": rows, "cols": cols, "n_z": n_z, "p": rng.choice((0.05, 0.1, 0.2, 0.5, 0.9)),
                "residual": rng.random() < 0.5, "train": rng.random() < 0.5}
    if op in ("norm", "norm_e4m3"):
        cols = _log(rng, 1, 32768)
        rows = _log(rng, 1, max(1, min(100_000, 40_000_000 // cols)))
        case = {"op": op, "dtype": dtype, "rows": rows, "cols": cols, "residual": rng.random() < 0.5}
        return case if op == "norm_e4m3" else {**case, "train": rng.random() < 0.7}
    if op == "w4":
        dtype = rng.choice(("fp32", "bf16", "fp16", "e4m3"))
    return {"op": op, "dtype": dtype, "rows": _log(rng, 1, 64), "in": _log(rng, 64, 12000), "out": _log(rng, 1, 12000),
            "group": rng.choice((32, 64, 128)), "zero": rng.random() < 0.5, "gamma": op == "w4" and rng.random() < 0.3}


def work(case):
    op, s = case["op"], _SIZE[case["dtype"]]
    if op == "dropout":
        n_in, n_out = case["rows"] * case["cols"], case["rows"] * case["n_z"] * case["cols"]
        b = s * (n_in + n_out + (n_out if case["residual"] else 0))
        if case["train"]:
            b += s * (n_out + n_in)
        return {"bytes": b, "flops": 2 * n_out * (2 if case["train"] else 1)}
    if op in ("norm", "norm_e4m3"):
        n, r = case["rows"] * case["cols"], case["residual"]
        b = n * (s * (3 if r else 1) + (1 if op == "norm_e4m3" else s)) + 4 * case["cols"]
        f = 5 * n
        if op == "norm_e4m3":
            b += 4 * case["rows"]
        elif case["train"]:          # the gradients of y and of h, h itself, the input's gradient, the weight and its gradient
            b += n * s * (4 if r else 3) + 8 * case["cols"]
            f += 9 * n
        return {"bytes": b, "flops": f}
    m, k, o = case["rows"], case["in"], case["out"]
    groups = -(-k // case["group"])
    b = o * k // 2 + o * groups * (5 if case["zero"] else 4) + 4 * o + (4 * o if case["gamma"] else 0)
    if op == "w4":
        b += m * k * s + m * o * (2 if case["dtype"] == "e4m3" else s) + (4 * m if case["dtype"] == "e4m3" else 0)
    else:
        b += m * k * s * 3 + 4 * k + m * o * s
    return {"bytes": b, "flops": 2 * m * k * o}


# ------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    rnd = lambda *shape: torch.randn(*shape, device=dev, generator=g)  # noqa: E731
    op = case["op"]
    st = {"case": case}
    if op == "dropout":
        dt = _DT[case["dtype"]]
        rows, cols, n_z = case["rows"], case["cols"], case["n_z"]
        shape = (rows, cols) if n_z == 1 else (rows, n_z, cols)
        st["x"] = rnd(rows, cols).to(dt)
        st["residual"] = rnd(*shape).to(dt) if case["residual"] else None
        st["seed"] = (seed * 0x9E3779B97F4A7C15 + 12345) & 0xFFFFFFFFFFFFFFFF
        # a multiple of four where a program shards whole batches, anything where rows of an odd width are sharded
        st["elem_offset"] = (seed % 1000) * cols * n_z
        if case["train"]:
            st["g"] = rnd(*shape).to(dt)
            st["x"].requires_grad_(True)
            if st["residual"] is not None:
                st["residual"].requires_grad_(True)
        return st
    if op in ("norm", "norm_e4m3", "norm_w4"):
        dt = _DT[case["dtype"]]
        rows, cols = case["rows"], case["in"] if op == "norm_w4" else case["cols"]
        st["x"] = rnd(rows, cols).to(dt)
        st["residual"] = (3 * rnd(rows, cols)).to(dt) if op == "norm_w4" or case["residual"] else None
        st["weight"] = 1 + 0.2 * rnd(cols)
        if op == "norm" and case["train"]:
            st["g"] = rnd(rows, cols).to(dt)
            st["gh"] = rnd(rows, cols).to(dt) if case["residual"] else None
            for k in ("x", "residual", "weight"):
                if st[k] is not None:
                    st[k].requires_grad_(True)
    if op in ("w4", "norm_w4"):
        m, k, o, group = case["rows"], case["in"], case["out"], case["group"]
        groups = -(-k // group)
        # bell-shaped 4-bit values, scales of a layer whose outputs are of order one
        st["q"] = (8 + 2.5 * rnd(o, k)).round_().clamp_(0, 15).to(torch.uint8)
        st["scale"] = (0.4 / k ** 0.5) * (0.5 + torch.rand(o, groups, device=dev, generator=g))
        st["zero"] = torch.randint(5, 11, (o, groups), device=dev, generator=g, dtype=torch.uint8) if case["zero"] else None
        st["bias"] = 0.1 * rnd(o)
        st["gamma"] = torch.rand(o, device=dev, generator=g) if case["gamma"] else None
        if op == "w4":
            x = rnd(m, k)
            if case["dtype"] == "e4m3":
                st["x_scale"] = x.abs().amax(1) / _E4M3_MAX
                st["x"] = (x / st["x_scale"][:, None]).to(torch.float8_e4m3fn)
            else:
                st["x_scale"], st["x"] = None, x.to(_DT[case["dtype"]])
        if own:          # weights are laid out once, when a program loads them
            import card_amd
            st["linear"] = card_amd.QuantLinear(st["q"], st["scale"], st["zero"], st["bias"], group=group)
    return st


# ------------------------------------------------------------------------------------------------------------ one pass
def run(st):
    return (_run_own if own else _run_plain)(st)


def _run_own(st):
    import card_amd
    case = st["case"]
    op = case["op"]
    if op == "dropout":
        y = card_amd.dropout(st["x"], case["p"], seed=st["seed"], elem_offset=st["elem_offset"], n_z=case["n_z"],
                             residual=st["residual"])
        if not case["train"]:
            return {"y": y}
        leaves = [st["x"]] + ([st["residual"]] if case["residual"] else [])
        grads = torch.autograd.grad(y, leaves, st["g"])
        return {"y": y, "dx": grads[0], **({"dresidual": grads[1]} if case["residual"] else {})}
    if op == "norm_e4m3":
        out = card_amd.rms_norm_e4m3(st["x"], st["weight"], residual=st["residual"])
        return dict(zip(("q", "scale", "h"), out))
    if op == "norm":
        if not case["residual"]:
            y = card_amd.rms_norm(st["x"], st["weight"])
            if not case["train"]:
                return {"y": y}
            dx, dw = torch.autograd.grad(y, (st["x"], st["weight"]), st["g"])
            return {"y": y, "dx": dx, "dweight": dw}
        y, h = card_amd.rms_norm(st["x"], st["weight"], residual=st["residual"])
        if not case["train"]:
            return {"y": y, "h": h}
        dx, dr, dw = torch.autograd.grad((y, h), (st["x"], st["residual"], st["weight"]), (st["g"], st["gh"]))
        return {"y": y, "h": h, "dx": dx, "dresidual": dr, "dweight": dw}
    if op == "w4":
        return {"y": st["linear"].forward(st["x"], st["x_scale"], gamma=st["gamma"], slope=0.01 if case["gamma"] else None)}
    q, scale, h = card_amd.rms_norm_e4m3(st["x"], st["weight"], residual=st["residual"])
    return {"h": h, "y": st["linear"].forward(q, scale, slope=0.01, out_dtype=_DT[case["dtype"]])}


def _philox_words(first_block, blocks, seed, device):
    """(blocks, 4) words of Philox4x32-10 for the counters (block lo, block hi, 0, 1); 32-bit values held in int64."""
    b = torch.arange(blocks, device=device, dtype=torch.int64) + first_block
    c0, c1, c2, c3 = b & _M32, (b >> 32) & _M32, torch.zeros_like(b), torch.ones_like(b)
    k0, k1 = seed & _M32, seed >> 32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57          # the low 64 bits are right, whatever the sign
        c0, c1, c2, c3 = ((p1 >> 32) & _M32) ^ c1 ^ k0, p1 & _M32, ((p0 >> 32) & _M32) ^ c3 ^ k1, p0 & _M32
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    return torch.stack((c0, c1, c2, c3), 1)


def _keep_plain(n, st):
    off, seed = st["elem_offset"], st["seed"]
    first, last = off // 4, (off + n - 1) // 4
    words = _philox_words(first, last - first + 1, seed, st["x"].device).reshape(-1)
    return words[off - 4 * first:][:n] >= round(st["case"]["p"] * 2 ** 32)


def _quant_rows(v):
    """e4m3 values of rows and the scale of each"""
    amax = v.abs().amax(-1, keepdim=True)
    return (v * (_E4M3_MAX / amax)).to(torch.float8_e4m3fn), (amax / _E4M3_MAX).squeeze(-1)


def _w4_plain(st, x):
    case = st["case"]
    o, k = st["q"].shape
    pad = -k % case["group"]
    zero = 8.0 if st["zero"] is None else st["zero"].float()[:, :, None]
    q = torch.nn.functional.pad(st["q"], (0, pad)).reshape(o, -1, case["group"]).float()
    w = ((q - zero) * st["scale"][:, :, None]).reshape(o, -1)[:, :k]
    return x @ w.t()


def _run_plain(st):
    with torch.no_grad():
        case = st["case"]
        op = case["op"]
        if op == "dropout":
            x, r = st["x"], st["residual"]
            rows, cols, n_z = case["rows"], case["cols"], case["n_z"]
            mask = _keep_plain(rows * n_z * cols, st).reshape(rows, n_z, cols)
            s = 1.0 / (1.0 - case["p"])
            y = torch.where(mask, x.float()[:, None, :] * s, 0.0)
            if r is not None:
                y = y + r.float().reshape(rows, n_z, cols)
            y = (y if n_z > 1 else y[:, 0]).to(x.dtype)
            if not case["train"]:
                return {"y": y}
            dx = torch.where(mask, st["g"].float().reshape(rows, n_z, cols) * s, 0.0).sum(1).to(x.dtype)
            return {"y": y, "dx": dx, **({"dresidual": st["g"]} if r is not None else {})}
        if op in ("norm", "norm_e4m3", "norm_w4"):
            x, r, w = st["x"], st["residual"], st["weight"]
            h = x.float() if r is None else x.float() + r.float()
            y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * w
            hs = {} if r is None else {"h": h.to(x.dtype)}
            if op == "norm_e4m3":
                q, scale = _quant_rows(y)
                return {"q": q, "scale": scale, **hs}
            if op == "norm":
                out = {"y": y.to(x.dtype), **hs}
                if case["train"]:
                    # in a row of a few values the two terms of dx all but cancel: 64 bits there
                    wide = torch.float64 if case["cols"] <= 16 else torch.float32
                    hb = h.to(x.dtype).to(wide)
                    rstd = torch.rsqrt(hb.square().mean(-1, keepdim=True) + 1e-6)
                    g = st["g"].to(wide)
                    gw = g * w
                    dx = rstd * gw - hb * (rstd.pow(3) * (gw * hb).mean(-1, keepdim=True))
                    if r is not None:
                        dx = dx + st["gh"].to(wide)
                    out["dx"] = dx.to(x.dtype)
                    if r is not None:
                        out["dresidual"] = out["dx"]
                    out["dweight"] = (g * hb * rstd).sum(0).float()
                return out
            q, scale = _quant_rows(y)
            out = _w4_plain(st, q.float() * scale[:, None]) + st["bias"]
            return {**hs, "y": torch.where(out > 0, out, 0.01 * out).to(_DT[case["dtype"]])}
        x = st["x"].float() if st["x_scale"] is None else st["x"].float() * st["x_scale"][:, None]
        y = _w4_plain(st, x) + st["bias"]
        if st["gamma"] is not None:
            y = y * st["gamma"]
            y = torch.where(y > 0, y, 0.01 * y)
        return {"y": y.to(torch.bfloat16 if case["dtype"] == "e4m3" else st["x"].dtype)}


# ------------------------------------------------------------------------------------------------------------ 64 bits
def _mul_hi_lo(a, m):
    """High and low words of the 64-bit product of a 32-bit tensor and a 32-bit constant, by 16-bit halves."""
    al, ah, ml, mh = a % 65536, a // 65536, m % 65536, m // 65536
    mid = ah * ml + (al * ml) // 65536
    cross = al * mh + mid % 65536
    return ah * mh + mid // 65536 + cross // 65536, (cross % 65536) * 65536 + (al * ml) % 65536


def _dropped_exact(n, st):
    """Whether each of n elements is dropped, from the generator's definition, in slices"""
    dev, out = st["x"].device, []
    for lo in range(0, n, 1 << 22):
        e = torch.arange(lo, min(n, lo + (1 << 22)), device=dev, dtype=torch.int64) + st["elem_offset"]
        block = e // 4
        c = [block % 2 ** 32, block // 2 ** 32, torch.zeros_like(e), torch.ones_like(e)]
        key = [st["seed"] % 2 ** 32, st["seed"] // 2 ** 32]
        for _ in range(10):
            h0, l0 = _mul_hi_lo(c[0], 0xD2511F53)
            h1, l1 = _mul_hi_lo(c[2], 0xCD9E8D57)
            c = [torch.bitwise_xor(torch.bitwise_xor(h1, c[1]), key[0]), l1, torch.bitwise_xor(torch.bitwise_xor(h0, c[3]), key[1]), l0]
            key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
        word = torch.stack(c).gather(0, (e % 4)[None])[0]
        out.append(word.double() / 2 ** 32 < round(st["case"]["p"] * 2 ** 32) / 2 ** 32)
    return torch.cat(out)


def exact(case, seed):
    st = prepare(case, seed)
    D = torch.float64
    op = case["op"]
    with torch.no_grad():
        if op == "dropout":
            rows, cols, n_z = case["rows"], case["cols"], case["n_z"]
            gone = _dropped_exact(rows * n_z * cols, st).reshape(rows, n_z, cols)
            x = st["x"].to(D).reshape(rows, 1, cols).expand(rows, n_z, cols)
            y = (x / (1 - case["p"])).masked_fill(gone, 0)
            if case["residual"]:
                y = y + st["residual"].to(D).reshape(rows, n_z, cols)
            out = {"y": y.reshape(st["residual"].shape if case["residual"] else (rows, cols) if n_z == 1 else y.shape)}
            if case["train"]:
                g = st["g"].to(D)
                out["dx"] = (g.reshape(rows, n_z, cols) / (1 - case["p"])).masked_fill(gone, 0).sum(1)
                if case["residual"]:
                    out["dresidual"] = g
            return out
        y = None
        if op in ("norm", "norm_e4m3", "norm_w4"):
            hid = st["x"].to(D)
            if st["residual"] is not None:
                hid = hid + st["residual"].to(D)
            norm = lambda h: h / ((h * h).sum(-1, keepdim=True) / h.shape[-1] + 1e-6).sqrt()  # noqa: E731
            y = norm(hid) * st["weight"].to(D)
            res = {} if st["residual"] is None else {"h": hid}
            if op == "norm_e4m3":
                top = y.abs().max(-1).values
                return {"q": y / top[:, None] * 448, "scale": top / 448, **res}
            if op == "norm":
                res = {"y": y, **res}
                if case["train"]:
                    # the backward pass starts from h as the forward pass stored it
                    h = (hid if st["residual"] is None else hid.to(st["x"].dtype).to(D))
                    g, w, n = st["g"].to(D), st["weight"].to(D), h.shape[-1]
                    unit, inv = norm(h), 1 / ((h * h).sum(-1, keepdim=True) / n + 1e-6).sqrt()
                    dx = inv * (g * w - unit * ((g * w * unit).sum(-1, keepdim=True) / n))
                    if st["gh"] is not None:
                        dx = dx + st["gh"].to(D)
                        res["dresidual"] = dx
                    res["dx"], res["dweight"] = dx, (g * unit).sum(0)
                return res
        if op == "w4":
            x = st["x"].to(D) if st["x_scale"] is None else st["x"].to(D) * st["x_scale"].to(D)[:, None]
        else:
            # the product sees rows of 8 bits: their rounding is part of the definition
            top = y.abs().max(-1, keepdim=True).values
            x = (y / top * 448).to(torch.float8_e4m3fn).to(D) * (top / 448)
        at = torch.arange(case["in"], device=x.device) // case["group"]
        parts = []
        for lo in range(0, case["out"], 4096):          # the weights in 64 bits, some rows at a time
            rows = slice(lo, lo + 4096)
            z = 8 if st["zero"] is None else st["zero"][rows].to(D)[:, at]
            parts.append(x @ ((st["q"][rows].to(D) - z) * st["scale"][rows].to(D)[:, at]).t())
        v = torch.cat(parts, 1) + st["bias"].to(D)
        if st["gamma"] is not None:
            v = v * st["gamma"].to(D)
        if op == "norm_w4" or st["gamma"] is not None:
            v = torch.nn.functional.leaky_relu(v, 0.01)
        return {"y": v, **({"h": hid} if op == "norm_w4" else {})}
