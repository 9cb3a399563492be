"""Cases that measure the engine's 8-bit serving operators.

Linear8: the product of tokens (rows, or the pixels of NCHW planes) with a weight matrix in 8-bit integers, a scale for
each token and each output channel, bias and SimpleGate in its ending; also straight from cached rows. RowCache: rows
quantised to 8 or 4 bits as they are written, and read back through page tables or row numbers.

`own` False runs the operators in elementary torch operations, `own` True runs the engine's kernels.
"""
import importlib
import math

import torch

own = False

TINY = 2.0 ** -126  # the smallest scale: a row of zeros has it


def _engine():
    from __graft_entry__ import load_package

    return importlib.import_module(load_package().__name__ + ".quant")


_DT = {"f16": torch.float16, "f32": torch.float32}
_BYTES = {"f16": 2, "f32": 4}


# ----------------------------------------------------------------------------------------------------------------------
# Cases
# ----------------------------------------------------------------------------------------------------------------------

def _linear(name, rows, k, n, x="f16", y="f16", gate=False, bias=True, planes=0):
    """planes: 0 token rows, else the number of images, rows pixels in all."""
    return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "x": x, "y": y, "gate": gate, "bias": bias,
            "planes": planes}


def _cached(name, frames, rows, cols, n, y="f16", gate=False, bias=True):
    return {"name": name, "op": "cached", "frames": frames, "rows": rows, "cols": cols, "n": n, "y": y, "gate": gate,
            "bias": bias}


def _append(name, rows, cols, capacity, bits=8, group=0, x="f16"):
    return {"name": name, "op": "append", "rows": rows, "cols": cols, "capacity": capacity, "bits": bits,
            "group": group, "x": x}


def _window(name, batch, page_rows, pages, cols, bits=8, group=0, y="f16"):
    return {"name": name, "op": "window", "batch": batch, "page_rows": page_rows, "pages": pages, "cols": cols,
            "bits": bits, "group": group, "y": y}


def listed():
    return [
        # One token through a hidden layer of the deepest level's width: the latency of a single call.
        _linear("one_token", 1, 512, 1024),
        # A handful of tokens with odd sizes, FP32 in and out.
        _linear("few_tokens_odd_f32", 13, 1000, 520, x="f32", y="f32"),
        # The gated expansion (conv4) of the middle level of a 1080p frame.
        _linear("middle_gated", 8160, 512, 1024, gate=True),
        # A 1x1 convolution 32 -> 64 over a 1080p frame in the public NCHW layout.
        _linear("planes_1080p", 1080 * 1920, 32, 64, planes=1),
        # The same kind of layer one level down, as token rows.
        _linear("level1_rows", 544 * 960, 64, 128),
        # A large square product: the compute-bound end.
        _linear("large_square", 8192, 4096, 4096),
        # The temporal fusion (5 frames x 64 channels -> 64) of level 1 read straight from the cache.
        _cached("fusion_level1", 5, 544 * 960, 64, 64),
        # The same at an odd crop and width.
        _cached("fusion_odd", 3, 1003, 96, 100, y="f32"),
        # Decoding: one new row for each of 64 sequences at scattered places of a long cache, and read back.
        _append("append_64", 64, 1024, 1 << 20),
        # A whole level-0 frame quantised into the cache and read back.
        _append("frame_level0", 1088 * 1920, 32, 2 * 1088 * 1920),
        # Five frames of level 1 read back.
        _window("window_level1", 1, 544 * 960, 5, 64),
        # Ragged sequences over small pages held in 4 bits with groups of 32.
        _window("ragged_4bit", 7, 16, 150, 512, bits=4, group=32, y="f32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "cached", "append", "window"])
    if op == "linear":
        k, n = _log(rng, 16, 4096), 2 * _log(rng, 4, 2048)
        most = min(2_000_000, int(8192 * 4096 * 4096 // (k * n)), int(100_000_000 // (k + n)))
        rows = _log(rng, 1, most)
        planes = rng.choice([0, 0, 1, 2]) if rows >= 64 else 0
        if planes == 2:
            rows -= rows % 2
        return dict(_linear("", rows, k, n, rng.choice(["f16", "f16", "f32"]) if not planes else "f16",
                            rng.choice(["f16", "f16", "f32"]) if not planes else "f16", rng.random() < 0.4,
                            rng.random() < 0.7, planes), name="drawn")
    if op == "cached":
        frames, cols, n = rng.randint(1, 7), _log(rng, 16, 512), 2 * _log(rng, 8, 256)
        rows = _log(rng, 1, min(500_000, int(100_000_000 // (frames * cols + n))))
        return dict(_cached("", frames, rows, cols, n, rng.choice(["f16", "f32"]), rng.random() < 0.4,
                            rng.random() < 0.7), name="drawn")
    bits = rng.choice([8, 4])
    group = rng.choice([0, 32, 64])
    cols = _log(rng, 16, 2048)
    if group:
        cols = max(group, cols - cols % group)
    if op == "append":
        rows = _log(rng, 1, min(1_000_000, int(60_000_000 // cols)))
        return dict(_append("", rows, cols, rows + _log(rng, 1, rows + 100), bits, group, rng.choice(["f16", "f32"])),
                    name="drawn")
    page_rows, batch = _log(rng, 1, 4096), rng.randint(1, 9)
    pages = _log(rng, 1, max(1, min(4096, int(60_000_000 // (cols * page_rows * batch)))))
    return dict(_window("", batch, page_rows, pages, cols, bits, group, rng.choice(["f16", "f32"])), name="drawn")


# ----------------------------------------------------------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _features(g, rows, cols, dtype):
    """Features as the layers meet them: every row with a level of its own, some channels far above the others."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x *= torch.exp(0.7 * torch.randn(rows, 1, generator=g, device="cuda"))
    x *= 1 + 7 * (torch.rand(1, cols, generator=g, device="cuda") > 0.95)
    return x.to(dtype)


def _pages(case, g):
    """A page table (batch, pages) over twice as many pages, no page twice, and the sequences' lengths."""
    b, n, p = case["batch"], case["pages"], case["page_rows"]
    table = torch.randperm(2 * b * n, generator=g, device="cuda")[: b * n].reshape(b, n).to(torch.int32)
    most = n * p
    if b == 1:
        return table, torch.full((1,), most, dtype=torch.int32, device="cuda")
    return table, (torch.rand(b, generator=g, device="cuda") * (most + 1)).to(torch.int32).clamp(max=most)


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    op = case["op"]
    if op in ("linear", "cached"):
        k = case["k"] if op == "linear" else case["frames"] * case["cols"]
        n = case["n"]
        s["w"] = (torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)).half()
        s["b"] = (0.1 * torch.randn(n, generator=g, device="cuda")).half() if case["bias"] else None
        s["wq"], s["ws"] = _quantise(s["w"], 8, k)
    if op == "linear":
        x = _features(g, case["rows"], case["k"], _DT[case["x"]])
        if case["planes"]:
            i = case["planes"]
            x = x.reshape(i, case["rows"] // i, case["k"]).transpose(1, 2).contiguous()
            side = 1920 if x.shape[2] % 1920 == 0 else 1
            x = x.reshape(i, case["k"], x.shape[2] // side, side)
        s["x"] = x
    elif op == "cached":
        # Twice as many frames are held as one window reads; the window takes every other one.
        x = _features(g, 2 * case["frames"] * case["rows"], case["cols"], torch.float16)
        s["pages"] = list(range(1, 2 * case["frames"], 2))
        _hold(s, x, 2 * case["frames"], case["rows"], case["cols"], 8, 0)
    elif op == "append":
        s["x"] = _features(g, case["rows"], case["cols"], _DT[case["x"]])
        s["out"] = torch.zeros(case["rows"], case["cols"], dtype=_DT[case["x"]], device="cuda")
        s["slots"] = torch.randperm(case["capacity"], generator=g, device="cuda")[: case["rows"]]
        if case["rows"] > 100_000:  # a frame: consecutive rows
            s["slots"] = torch.arange(case["rows"], device="cuda") + (case["capacity"] - case["rows"])
        s["first"] = case["capacity"] - case["rows"] if case["rows"] > 100_000 else None
        _hold(s, None, case["capacity"], 1, case["cols"], case["bits"], case["group"])
    else:
        s["table"], s["lengths"] = _pages(case, g)
        most = case["pages"] * case["page_rows"]
        s["out"] = torch.zeros(case["batch"], most, case["cols"], dtype=_DT[case["y"]], device="cuda")
        total = 2 * case["batch"] * case["pages"]
        _hold(s, _features(g, total * case["page_rows"], case["cols"], torch.float16), total, case["page_rows"],
              case["cols"], case["bits"], case["group"])
    if own:
        if op in ("linear", "cached"):
            s["layer"] = _engine().Linear8.from_tensors(s["w"], s["b"], gate=case["gate"],
                                                        segments=case["frames"] if op == "cached" else 1)
    return s


def _hold(s, x, pages, page_rows, cols, bits, group):
    """The cache that a program holds: the engine's, or its codes (one for a byte) and scales as tensors."""
    if own:
        s["cache"] = _engine().RowCache(pages, page_rows, cols, bits=bits, group=group)
        if x is not None:
            s["cache"].write(x)
    elif x is not None:
        s["q"], s["s"] = _quantise(x, bits, group or cols)
    else:
        s["q"] = torch.zeros(pages * page_rows, cols, dtype=torch.int8, device="cuda")
        s["s"] = torch.zeros(pages * page_rows, cols // (group or cols), device="cuda")


# ----------------------------------------------------------------------------------------------------------------------
# The plain forms
# ----------------------------------------------------------------------------------------------------------------------

def _quantise(x, bits, group):
    """Codes and scales of the groups of x's rows: s = max |x| / qmax, the code the nearest whole number to x / s. The
    quotient is taken in 64 bits, so that one next to the border of two codes falls on the right side."""
    q = 127 if bits == 8 else 7
    v = x.float().reshape(x.shape[0], -1, group)
    a = v.abs().amax(2, keepdim=True)
    fine = torch.isfinite(a)
    s = torch.where(fine, (a / q).clamp_min(TINY), float("nan"))
    codes = torch.where(fine, (v.double() / s.double()).round(), 0.0).to(torch.int8)
    return codes.reshape(x.shape), s.reshape(x.shape[0], -1)


def _finish(acc, case, bias):
    if bias is not None:
        acc = acc + bias.float()
    if case["gate"]:
        h = case["n"] // 2
        acc = acc[:, :h] * acc[:, h:]
    return acc


def _plain(s):
    case, op = s["case"], s["case"]["op"]
    if op == "linear":
        x = s["x"]
        if case["planes"]:
            x = x.flatten(2).transpose(1, 2).reshape(case["rows"], case["k"])
        q, sx = _quantise(x, 8, case["k"])
        y = _finish((q.float() @ s["wq"].float().t()) * sx * s["ws"].t(), case, s["b"]).to(_DT[case["y"]])
        if case["planes"]:
            i, _, h, w = s["x"].shape
            y = y.reshape(i, h * w, -1).transpose(1, 2).reshape(i, -1, h, w).contiguous()
        return y
    if op == "cached":
        r = case["rows"]
        x = (s["q"].reshape(-1, r, case["cols"])[s["pages"]].float() * s["s"].reshape(-1, r, 1)[s["pages"]])
        x = x.transpose(0, 1).reshape(r, -1)
        return _finish((x @ s["wq"].float().t()) * s["ws"].t(), case, s["b"]).to(_DT[case["y"]])
    group = case["group"] or case["cols"]
    if op == "append":
        q, sx = _quantise(s["x"], case["bits"], group)
        s["q"][s["slots"]], s["s"][s["slots"]] = q, sx
        q, sx = s["q"][s["slots"]], s["s"][s["slots"]]
        s["out"].copy_((q.float().reshape(case["rows"], -1, group) * sx[:, :, None]).reshape(case["rows"], -1))
        return s["out"]
    p, most = case["page_rows"], case["pages"] * case["page_rows"]
    at = (s["table"].long()[:, :, None] * p + torch.arange(p, device="cuda")).reshape(case["batch"], most)
    live = torch.arange(most, device="cuda")[None] < s["lengths"][:, None]
    v = s["q"][at].float().reshape(case["batch"], most, -1, group) * s["s"][at][..., None]
    s["out"].copy_(torch.where(live[:, :, None], v.reshape(s["out"].shape), s["out"].float()))
    return s["out"]


def run(state):
    if not own:
        return _plain(state)
    case, op = state["case"], state["case"]["op"]
    if op == "linear":
        if case["planes"]:
            return state["layer"].forward_nchw(state["x"])
        return state["layer"].forward(state["x"], out_dtype=_DT[case["y"]])
    if op == "cached":
        return state["layer"].forward_cached(state["cache"], state["pages"], out_dtype=_DT[case["y"]])
    if op == "append":
        if state["first"] is not None:
            state["cache"].write(state["x"], row0=state["first"])
        else:
            state["cache"].write(state["x"], slots=state["slots"])
        return state["cache"].read_rows(state["slots"], out=state["out"])
    return state["cache"].read(state["table"], state["lengths"], out=state["out"])


# ----------------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ----------------------------------------------------------------------------------------------------------------------

def _held(case, rows):
    """Bytes of `rows` cached rows: codes and scales."""
    return rows * ((case["cols"] * case["bits"] + 7) // 8 + 4 * (case["cols"] // (case["group"] or case["cols"])))


def work(case):
    op = case["op"]
    if op == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": rows * k * _BYTES[case["x"]] + n * (k + 4 + 2 * case["bias"]) +
                rows * (n // 2 if case["gate"] else n) * _BYTES[case["y"]], "flops": 2 * rows * k * n}
    if op == "cached":
        rows, n, t, c = case["rows"], case["n"], case["frames"], case["cols"]
        return {"bytes": rows * t * (c + 4) + n * (t * c + 4 + 2 * case["bias"]) +
                rows * (n // 2 if case["gate"] else n) * _BYTES[case["y"]], "flops": 2 * rows * t * c * n}
    if op == "append":
        rows, cols = case["rows"], case["cols"]
        return {"bytes": 2 * rows * cols * _BYTES[case["x"]] + 2 * _held(case, rows) + 8 * rows, "flops": 4 * rows * cols}
    rows = case["batch"] * case["pages"] * case["page_rows"]
    rows = rows if case["batch"] == 1 else rows // 2  # the lengths are spread evenly
    return {"bytes": _held(case, rows) + rows * case["cols"] * _BYTES[case["y"]], "flops": rows * case["cols"]}


# ----------------------------------------------------------------------------------------------------------------------
# The same in 64 bits, from the definition
# ----------------------------------------------------------------------------------------------------------------------

def _values64(x, qmax, group):
    """The values that the nearest codes stand for, in 64 bits. The scale is the 32-bit quotient of the group's largest
    magnitude and qmax: that rounding is part of the definition."""
    v = x.double().unflatten(1, (-1, group))
    top = torch.linalg.vector_norm(v, float("inf"), dim=2, keepdim=True)
    scale = torch.maximum((top.float() / qmax), torch.tensor(TINY, device=x.device)).double()
    low = torch.floor(v / scale)
    over = v / scale - low  # nearest, halves to the even neighbour
    code = low + ((over > 0.5) | ((over == 0.5) & (low.remainder(2) == 1))).double()
    return (code * scale).flatten(1)


def exact(case, seed):
    global own
    kept, own = own, False
    s = prepare(case, seed)
    own = kept
    op = case["op"]
    if op in ("linear", "cached"):
        w = _values64(s["w"], 127, s["w"].shape[1])
    # The source rows are made again: the cache's own content comes from them.
    g = _gen(seed)
    if op in ("linear", "cached"):
        torch.randn(s["w"].shape, generator=g, device="cuda")
        if case["bias"]:
            torch.randn(case["n"], generator=g, device="cuda")
    if op == "linear":
        x = s["x"].flatten(2).movedim(1, 2).flatten(0, 1) if case["planes"] else s["x"]
        v = _values64(x, 127, case["k"])
    elif op == "cached":
        x = _features(g, 2 * case["frames"] * case["rows"], case["cols"], torch.float16)
        x = x.unflatten(0, (-1, case["rows"]))
        v = torch.cat([_values64(x[p], 127, case["cols"]) for p in s["pages"]], 1)
    else:
        qmax, group = (127 if case["bits"] == 8 else 7), case["group"] or case["cols"]
        if op == "append":
            return _values64(s["x"], qmax, group)
        _pages(case, g)
        total = 2 * case["batch"] * case["pages"]
        x = _features(g, total * case["page_rows"], case["cols"], torch.float16).unflatten(0, (total, -1))
        want = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["lengths"].tolist()):
            rows = x[s["table"][b].long()].flatten(0, 1)[:n]
            if n:
                want[b, :n] = _values64(rows, qmax, group)
        return want
    y = torch.einsum("mk,nk->mn", v, w)
    if s["b"] is not None:
        y += s["b"].double()
    if case["gate"]:
        a, b = y.chunk(2, 1)
        y = a * b
    if op == "linear" and case["planes"]:
        i, _, h, w2 = s["x"].shape
        y = y.unflatten(0, (i, h, w2)).permute(0, 3, 1, 2).contiguous()
    return y
