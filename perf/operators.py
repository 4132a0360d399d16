"""What is measured of the sparse joint-attention path: positions to rotation
tables, the Q/K norm with the rotation from positions, the block means, the
block lists and the attention over them. Every case runs in a plain form
(elementary torch operations) and, with ``own`` set, through the library."""
import math

import torch

own = False

D = 128
TWO_PI = 2.0 * math.pi


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # One text + image sequence of 256 x 256 pixels (256 image, 512 caption tokens, 30 heads): latency.
        dict(name="prologue-256px", op="prologue", frames=1, height=16, width=16, text=512, heads=30, kv_heads=30,
             axes="32,48,48", theta=256.0, one_progression=False, t_scale=1.0, split_half=False, norm=True, fused=True),
        # The multi-reference sequence: 512 text tokens, 64 x 64 image tokens and three references, 32 heads.
        dict(name="prologue-multiref", op="prologue", frames=4, height=64, width=64, text=512, heads=32, kv_heads=32,
             axes="32,32,32,32", theta=10000.0, one_progression=False, t_scale=1.0, split_half=False, norm=True, fused=True),
        # A video clip of odd sizes, shared key heads, one frequency progression, halves paired, rotation only.
        dict(name="rotation-video-odd", op="prologue", frames=13, height=45, width=53, text=0, heads=30, kv_heads=6,
             axes="32,48,48", theta=10000.0, one_progression=True, t_scale=2.5, split_half=True, norm=False, fused=False),
        # Tables of one 1024 x 1024 pixel image with its text, for the projections that rotate in their epilogue.
        dict(name="tables-1024px", op="tables", frames=1, height=64, width=64, text=512, axes="32,32,32,32", theta=2000.0,
             one_progression=False, t_scale=1.0, head_dim=128),
        # Tables of a long clip: 33 frames of 60 x 68 tokens.
        dict(name="tables-video", op="tables", frames=33, height=60, width=68, text=226, axes="32,48,48", theta=10000.0,
             one_progression=False, t_scale=0.625, head_dim=128),
        # Block means of one 1024 x 1024 pixel sequence.
        dict(name="means-1024px", op="means", seq=4608, heads=30, block=64, masked=False),
        # The same for a long sequence of odd length with padded rows.
        dict(name="means-multiref-odd", op="means", seq=16889, heads=32, block=128, masked=True),
        # Lists for one new row against a long cache, shared key heads.
        dict(name="select-one-row", op="select", q_blocks=1, k_blocks=2048, heads=32, kv_heads=8, topk=64, keep_first=1,
             keep_last=2, empty=0.02),
        # Lists for the multi-reference sequence: 128-row query blocks, 64-row key blocks, the text always kept.
        dict(name="select-multiref", op="select", q_blocks=132, k_blocks=264, heads=32, kv_heads=32, topk=64, keep_first=8,
             keep_last=0, empty=0.0),
        # One row over 64 blocks of a cache of 65 536 rows, shared key heads.
        dict(name="attention-one-row", op="attention", seq_q=1, seq_k=65536, heads=32, kv_heads=8, q_block=1, k_block=64,
             list_len=64, masked=False, short=0.0),
        # Odd length, padded rows, lists that are not full.
        dict(name="attention-1024px-odd", op="attention", seq_q=4333, seq_k=4333, heads=30, kv_heads=30, q_block=128,
             k_block=64, list_len=18, masked=True, short=0.1),
        # The multi-reference sequence over a quarter of its keys.
        dict(name="attention-multiref", op="attention", seq_q=16896, seq_k=16896, heads=32, kv_heads=32, q_block=128,
             k_block=64, list_len=64, masked=False, short=0.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng, most):
    kv = _log(rng, 1, most)
    return kv * rng.randint(1, max(1, min(8, most // kv))), kv


def draw(rng):
    op = rng.choice(["prologue", "tables", "means", "select", "attention", "attention"])
    axes = rng.choice(["32,48,48", "32,32,32,32", "16,56,56", "64,64", "44,42,42", "128", "24,40,40"])
    place = dict(frames=rng.choice([1, 1, 2, _log(rng, 1, 24)]), height=_log(rng, 1, 48), width=_log(rng, 1, 48),
                 text=rng.choice([0, 1, _log(rng, 1, 512), 512]), axes=axes,
                 theta=rng.choice([256.0, 2000.0, 10000.0, 1.0e6]), one_progression=rng.random() < 0.3,
                 t_scale=rng.choice([1.0, 1.0, 0.625, 2.5, 24.0]))
    if op == "prologue":
        rows = place["frames"] * place["height"] * place["width"] + place["text"]
        heads, kv = _heads(rng, max(1, min(40, 500000 // rows)))
        return dict(op=op, heads=heads, kv_heads=kv, split_half=rng.random() < 0.4, norm=rng.random() < 0.8,
                    fused=rng.random() < 0.7, **place)
    if op == "tables":
        return dict(op=op, head_dim=128, **place)
    if op == "means":
        seq = _log(rng, 1, 16896)
        return dict(op=op, seq=seq, heads=rng.randint(1, 32), block=rng.choice([16, 32, 64, 128, 256, _log(rng, 1, 512)]),
                    masked=rng.random() < 0.5)
    if op == "select":
        heads, kv = _heads(rng, 32)
        k_blocks = _log(rng, 1, 2048)
        q_blocks = _log(rng, 1, max(1, min(132, 34848 // k_blocks)))
        return dict(op=op, q_blocks=q_blocks, k_blocks=k_blocks, heads=heads, kv_heads=kv,
                    topk=_log(rng, 4, 128), keep_first=rng.randint(0, 2), keep_last=rng.randint(0, 2),
                    empty=rng.choice([0.0, 0.0, 0.1, 0.9]))
    heads, kv = _heads(rng, 32)
    q_block, k_block = rng.choice([(1, 64), (128, 64), (128, 128), (256, 64), (128, 32), (64, 64), (384, 256), (100, 16)])
    one = rng.random() < 0.3
    q_block = 1 if one else max(16, q_block)
    seq_q = rng.randint(1, 4) if one else _log(rng, 2, 16896)
    seq_k = _log(rng, 1, 65536) if one else max(1, seq_q + rng.randint(-min(seq_q - 1, 77), 300))
    k_blocks = (seq_k + k_block - 1) // k_block
    most = min(k_blocks, max(1, 4096 // k_block))
    if not one:   # rows of the query tiles x listed keys x heads: at most half of the largest listed case
        tiles = (seq_q + q_block - 1) // q_block * ((q_block + 127) // 128) * 128
        most = max(1, min(most, 16896 * 4096 * 16 // (tiles * k_block * heads)))
    return dict(op="attention", seq_q=seq_q, seq_k=seq_k, heads=heads, kv_heads=kv, q_block=q_block, k_block=k_block,
                list_len=_log(rng, 1, most), masked=rng.random() < 0.5, short=rng.choice([0.0, 0.0, 0.3]))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _axes(case):
    return [int(a) for a in case["axes"].split(",")]


def _positions(case):
    """[seq, n] int32: text rows count along the last axis (or the first, with
    three axes and fewer), then the frames of the clip row by row; the last of
    four axes is the text's, as in the four-axis image models."""
    n, text = len(_axes(case)), case["text"]
    f, h, w = case["frames"], case["height"], case["width"]
    t = torch.arange(f, device="cuda").view(f, 1, 1).expand(f, h, w).reshape(-1)
    y = torch.arange(h, device="cuda").view(1, h, 1).expand(f, h, w).reshape(-1)
    x = torch.arange(w, device="cuda").view(1, 1, w).expand(f, h, w).reshape(-1)
    pos = torch.zeros(text + f * h * w, n, device="cuda", dtype=torch.int32)
    ids = torch.arange(text, device="cuda", dtype=torch.int32)
    if n == 4:
        pos[:text, 3] = ids
        pos[text:, 0], pos[text:, 1], pos[text:, 2] = 10 * t, y, x
        pos[text:, 3] = -t
    else:
        pos[:text, 0] = ids
        if n == 1:
            pos[text:, 0] = text + (t * h + y) * w + x
        elif n == 2:
            pos[text:, 0], pos[text:, 1] = text + t * h + y, x
        else:
            pos[text:, 0], pos[text:, 1], pos[text:, 2] = text + t, y, x
    return pos


def _scales(case):
    return [case["t_scale"]] + [1.0] * (len(_axes(case)) - 1)


def _library():
    import __graft_entry__
    lib = __graft_entry__.load_package().load()
    lib.init()
    return lib


def _row_mask(gen, rows, holes=0.02):
    """int32 [rows]: padding behind the last tenth and a few holes."""
    mask = (torch.rand(rows, generator=gen, device="cuda") >= holes).int()
    mask[max(1, rows - rows // 10):] = 0
    return mask


def _blocks(rows, block):
    return (rows + block - 1) // block


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=case)
    if own:
        s["lib"] = _library()
    op = case["op"]
    if op in ("prologue", "tables"):
        s["pos"] = _positions(case)
        if own:
            s["axes"] = s["lib"].rope_axes(_axes(case), _scales(case), case["theta"], case["one_progression"], D)
    if op == "prologue":
        seq, hq, hk = s["pos"].shape[0], case["heads"] * D, case["kv_heads"] * D
        # The projection's output rows hold Q, K and V (fused), or Q and K only.
        s["x"] = (_randn(gen, seq, hq + hk * (2 if case["fused"] else 1)) * 1.5).bfloat16()
        s["wq"] = 1.0 + 0.2 * _randn(gen, D)
        s["wk"] = 1.0 + 0.2 * _randn(gen, D)
        s["q_out"] = torch.empty(seq, hq, device="cuda", dtype=torch.bfloat16)
        s["k_out"] = torch.empty(seq, hk, device="cuda", dtype=torch.bfloat16)
    elif op == "tables":
        # Every seed stands at another place of a long clip.
        s["pos"] = s["pos"] + torch.tensor([seed % 997], device="cuda", dtype=torch.int32)
        s["cos"] = torch.empty(s["pos"].shape[0], case["head_dim"] // 2, device="cuda")
        s["sin"] = torch.empty_like(s["cos"])
    elif op == "means":
        n = _blocks(case["seq"], case["block"])
        s["x"] = (_randn(gen, case["seq"], case["heads"] * D) + 0.3 * _randn(gen, 1, case["heads"] * D)).bfloat16()
        s["mask"] = _row_mask(gen, case["seq"]) if case["masked"] else None
        s["means"] = torch.empty(n, case["heads"], D, device="cuda")
        s["counts"] = torch.empty(n, device="cuda", dtype=torch.int32)
    elif op == "select":
        s["qm"] = 0.3 * _randn(gen, case["q_blocks"], case["heads"], D)
        s["km"] = 0.3 * _randn(gen, case["k_blocks"], case["kv_heads"], D)
        s["counts"] = torch.randint(1, 65, (case["k_blocks"],), generator=gen, device="cuda", dtype=torch.int32)
        s["counts"][torch.rand(case["k_blocks"], generator=gen, device="cuda") < case["empty"]] = 0
        s["list"] = torch.empty(case["heads"], case["q_blocks"], case["topk"], device="cuda", dtype=torch.int32)
    else:
        nq, nk = _blocks(case["seq_q"], case["q_block"]), _blocks(case["seq_k"], case["k_block"])
        s["q"] = _randn(gen, case["seq_q"], case["heads"] * D).bfloat16()
        kv = _randn(gen, case["seq_k"], 2 * case["kv_heads"] * D).bfloat16()
        s["k"], s["v"] = kv[:, :case["kv_heads"] * D], kv[:, case["kv_heads"] * D:]
        s["mask"] = _row_mask(gen, case["seq_k"]) if case["masked"] else None
        # Distinct blocks in ascending order; a share of the lists is not full.
        order = torch.rand(case["heads"], nq, nk, generator=gen, device="cuda").argsort(dim=2)[:, :, :case["list_len"]]
        keep = torch.randint(0, case["list_len"] + 1, (case["heads"], nq, 1), generator=gen, device="cuda")
        full = torch.rand(case["heads"], nq, 1, generator=gen, device="cuda") >= case["short"]
        order = torch.where(full | (torch.arange(order.shape[2], device="cuda") < keep), order, nk).sort(dim=2)[0]
        s["list"] = torch.where(order < nk, order, -1).int().contiguous()
        s["out"] = torch.empty(case["seq_q"], case["heads"] * D, device="cuda", dtype=torch.bfloat16)
        s["scale"] = 1.0 / math.sqrt(D)
    return s


# ---------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------

def _angles(case, pos, head_dim):
    """[seq, head_dim / 2] angles in 64 bits."""
    half, cols, j = head_dim // 2, [], 0
    for a, (dim, scale) in enumerate(zip(_axes(case), _scales(case))):
        for i in range(dim // 2):
            power = -2.0 * j / head_dim if case["one_progression"] else -2.0 * i / dim
            cols.append((a, scale * case["theta"] ** power))
            j += 1
    axis = torch.tensor([a for a, _ in cols] + [0] * (half - j), device=pos.device)
    freq = torch.tensor([f for _, f in cols] + [0.0] * (half - j), device=pos.device, dtype=torch.float64)
    return pos[:, axis].double() * freq


def _plain_prologue(s):
    case = s["case"]
    hq, hk = case["heads"], case["kv_heads"]
    angle = _angles(case, s["pos"], D)
    cos, sin = angle.cos().float().unsqueeze(1), angle.sin().float().unsqueeze(1)

    def one(x, heads, w):
        x = x.float().reshape(x.shape[0], heads, D)
        if case["norm"]:
            x = x * (x.square().mean(2, keepdim=True) + 1e-6).rsqrt() * w
        if case["split_half"]:
            a, b = x[..., :D // 2], x[..., D // 2:]
            y = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=2)
        else:
            a, b = x[..., 0::2], x[..., 1::2]
            y = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=3)
        return y.reshape(x.shape[0], heads * D).bfloat16()

    return one(s["x"][:, :hq * D], hq, s["wq"]), one(s["x"][:, hq * D:(hq + hk) * D], hk, s["wk"])


def _plain_means(s):
    case = s["case"]
    seq, block, heads = case["seq"], case["block"], case["heads"]
    n = _blocks(seq, block)
    x = torch.zeros(n * block, heads * D, device="cuda", dtype=torch.float64)
    x[:seq] = s["x"].double()
    valid = torch.zeros(n * block, device="cuda", dtype=torch.bool)
    valid[:seq] = True if s["mask"] is None else s["mask"] != 0
    x = torch.where(valid.unsqueeze(1), x, 0.0).reshape(n, block, heads, D)
    counts = valid.reshape(n, block).sum(1)
    return (x.sum(1) / counts.clamp(min=1).view(n, 1, 1)).float(), counts.int()


def _plain_select(s):
    case = s["case"]
    group, nk, topk = case["heads"] // case["kv_heads"], case["k_blocks"], case["topk"]
    k = s["km"].double().repeat_interleave(group, dim=1)
    score = torch.matmul(s["qm"].double().permute(1, 0, 2), k.permute(1, 2, 0))
    j = torch.arange(nk, device="cuda")
    kept = (j < case["keep_first"]) | (j >= nk - case["keep_last"])
    score = score.masked_fill(kept, math.inf).masked_fill(s["counts"] == 0, -math.inf)
    best = score.sort(dim=2, descending=True, stable=True)[1][:, :, :topk]
    best = torch.where(s["counts"][best] > 0, best, nk).sort(dim=2)[0]
    out = torch.full((case["heads"], case["q_blocks"], topk), -1, device="cuda", dtype=torch.int32)
    out[:, :, :best.shape[2]] = torch.where(best < nk, best, -1).int()
    return out


def _plain_attention(s):
    case = s["case"]
    heads, group = case["heads"], case["heads"] // case["kv_heads"]
    qb, kb, seq_q, seq_k = case["q_block"], case["k_block"], case["seq_q"], case["seq_k"]
    nq, nk = _blocks(seq_q, qb), _blocks(seq_k, kb)
    valid = torch.zeros(nk * kb, device="cuda", dtype=torch.bool)
    valid[:seq_k] = True if s["mask"] is None else s["mask"] != 0
    valid = valid.reshape(nk, kb)

    def padded(x, h, rows):
        y = torch.zeros(rows, D, device="cuda", dtype=torch.float32)
        y[:x.shape[0]] = x[:, h * D:(h + 1) * D].float()
        return y

    outs = []
    for h in range(heads):
        q = padded(s["q"], h, nq * qb).reshape(nq, qb, D)
        if h % group == 0:
            k = padded(s["k"], h // group, nk * kb).reshape(nk, kb, D)
            v = padded(s["v"], h // group, nk * kb).reshape(nk, kb, D)
        index = s["list"][h].long()
        ok = ((index >= 0).unsqueeze(2) & valid[index.clamp(min=0)]).reshape(nq, 1, -1)
        index = index.clamp(min=0)
        score = torch.matmul(q, k[index].reshape(nq, -1, D).transpose(1, 2)) * s["scale"]
        score = score.masked_fill(~ok, -math.inf)
        top = score.amax(2, keepdim=True)
        p = (score - torch.where(top == -math.inf, 0.0, top)).exp()
        total = p.sum(2, keepdim=True)
        out = torch.matmul(p, v[index].reshape(nq, -1, D)) / torch.where(total == 0.0, 1.0, total)
        outs.append(out.reshape(nq * qb, D)[:seq_q].bfloat16())
    return torch.cat(outs, dim=1)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _own(s):
    case, lib, op = s["case"], s["lib"], s["case"]["op"]
    # 1 is CUDA's handle of the default stream; 0 would mean the library's own.
    lib.iris_b200_use_stream(torch.cuda.current_stream().cuda_stream or 1)
    if op == "prologue":
        x, hq, hk = s["x"].data_ptr(), case["heads"], case["kv_heads"]
        wq, wk = (s["wq"].data_ptr(), s["wk"].data_ptr()) if case["norm"] else (None, None)
        rc = lib.iris_b200_qk_norm_rope_axes(
            s["q_out"].data_ptr(), hq * D, s["k_out"].data_ptr(), hk * D, x, x + hq * D * 2, s["x"].shape[1], wq, wk,
            s["pos"].data_ptr(), s["axes"], s["x"].shape[0], hq, hk, D, 1e-6, int(case["split_half"]))
        out = s["q_out"], s["k_out"]
    elif op == "tables":
        rc = lib.iris_b200_rope_axes_tables(s["cos"].data_ptr(), s["sin"].data_ptr(), s["pos"].data_ptr(), s["axes"],
                                            s["pos"].shape[0], case["head_dim"])
        out = s["cos"], s["sin"]
    elif op == "means":
        rc = lib.iris_b200_block_means(s["means"].data_ptr(), s["counts"].data_ptr(), s["x"].data_ptr(), case["heads"] * D,
                                       case["seq"], case["heads"], D, case["block"],
                                       None if s["mask"] is None else s["mask"].data_ptr())
        out = s["means"], s["counts"]
    elif op == "select":
        rc = lib.iris_b200_block_select(s["list"].data_ptr(), s["qm"].data_ptr(), s["km"].data_ptr(), s["counts"].data_ptr(),
                                        case["q_blocks"], case["k_blocks"], case["heads"], case["kv_heads"], D,
                                        case["topk"], case["keep_first"], case["keep_last"])
        out = s["list"]
    else:
        rc = lib.iris_b200_attention_blocks(
            s["out"].data_ptr(), case["heads"] * D, s["q"].data_ptr(), case["heads"] * D, s["k"].data_ptr(),
            2 * case["kv_heads"] * D, s["v"].data_ptr(), 2 * case["kv_heads"] * D, case["seq_q"], case["seq_k"], case["heads"],
            case["kv_heads"], D, s["scale"], None if s["mask"] is None else s["mask"].data_ptr(), s["list"].data_ptr(), s["list"].shape[2],
            case["q_block"], case["k_block"], 0)
        out = s["out"]
    if rc:
        raise RuntimeError("iris_b200 error %d" % rc)
    return out


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "prologue":
        return _plain_prologue(state)
    if op == "tables":
        angle = _angles(state["case"], state["pos"], state["case"]["head_dim"])
        return angle.cos().float(), angle.sin().float()
    return {"means": _plain_means, "select": _plain_select, "attention": _plain_attention}[op](state)


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def _exact_turn(case, pos, head_dim):
    """e^(i angle) [seq, head_dim / 2], one pair at a time."""
    turn = torch.ones(pos.shape[0], head_dim // 2, device="cuda", dtype=torch.complex128)
    pair = 0
    for axis, dim in enumerate(_axes(case)):
        for i in range(dim // 2):
            base = pair / (head_dim // 2) if case["one_progression"] else i / (dim // 2)
            step = (case["t_scale"] if axis == 0 else 1.0) * math.exp(-math.log(case["theta"]) * base)
            turn[:, pair] = torch.polar(torch.ones((), device="cuda", dtype=torch.float64), pos[:, axis].double() * step)
            pair += 1
    return turn


def _exact_rows(x, heads, w, turn, case):
    x = x.double().reshape(x.shape[0], heads, D)
    if case["norm"]:
        x = x * w.double() / torch.sqrt((x * x).sum(-1, keepdim=True) / D + 1e-6)
    if case["split_half"]:
        z = torch.complex(x[..., :D // 2].contiguous(), x[..., D // 2:].contiguous()) * turn.unsqueeze(1)
        y = torch.cat((z.real, z.imag), dim=-1)
    else:
        y = torch.view_as_real(torch.view_as_complex(x.reshape(x.shape[0], heads, D // 2, 2).contiguous()) * turn.unsqueeze(1))
    return y.reshape(x.shape[0], heads * D)


def _exact_attention(case, s):
    out = torch.zeros(case["seq_q"], case["heads"] * D, device="cuda", dtype=torch.float64)
    lists = s["list"].cpu()
    usable = torch.ones(case["seq_k"], device="cuda", dtype=torch.bool) if s["mask"] is None else s["mask"].bool()
    rows = torch.arange(case["seq_k"], device="cuda")
    for h in range(case["heads"]):
        g = h * case["kv_heads"] // case["heads"]
        q = s["q"][:, h * D:(h + 1) * D].double()
        k, v = (s[n][:, g * D:(g + 1) * D].double() for n in "kv")
        for i in range(lists.shape[1]):
            mine = [rows[b * case["k_block"]:(b + 1) * case["k_block"]] for b in lists[h, i].tolist() if b >= 0]
            if not mine:
                continue
            keys = torch.cat(mine)
            keys = keys[usable[keys]]
            if not keys.numel():
                continue
            lo, hi = i * case["q_block"], min((i + 1) * case["q_block"], case["seq_q"])
            weight = torch.softmax(s["scale"] * (q[lo:hi] @ k[keys].T), dim=1)
            out[lo:hi, h * D:(h + 1) * D] = weight @ v[keys]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "prologue":
        turn = _exact_turn(case, s["pos"], D)
        hq, hk = case["heads"] * D, case["kv_heads"] * D
        return (_exact_rows(s["x"][:, :hq], case["heads"], s["wq"], turn, case),
                _exact_rows(s["x"][:, hq:hq + hk], case["kv_heads"], s["wk"], turn, case))
    if op == "tables":
        turn = _exact_turn(case, s["pos"], case["head_dim"])
        return turn.real.clone(), turn.imag.clone()
    if op == "means":
        valid = torch.ones(case["seq"], device="cuda", dtype=torch.float64) if s["mask"] is None else s["mask"].ne(0).double()
        block = torch.arange(case["seq"], device="cuda") // case["block"]
        n = _blocks(case["seq"], case["block"])
        counts = torch.zeros(n, device="cuda", dtype=torch.float64).index_add_(0, block, valid)
        sums = torch.zeros(n, case["heads"] * D, device="cuda", dtype=torch.float64)
        sums.index_add_(0, block, s["x"].double() * valid.unsqueeze(1))
        means = sums / counts.clamp(min=1.0).unsqueeze(1)
        return means.reshape(n, case["heads"], D), counts.int()
    if op == "select":
        out = torch.full((case["heads"], case["q_blocks"], case["topk"]), -1, dtype=torch.int32)
        counts = s["counts"].tolist()
        nk = case["k_blocks"]
        usable = [j for j in range(nk) if counts[j] > 0]
        always = [j for j in usable if j < case["keep_first"] or j >= nk - case["keep_last"]]
        others = [j for j in usable if j not in set(always)]
        room = case["topk"] - len(always)
        where = torch.tensor(others, device="cuda", dtype=torch.long)
        for h in range(case["heads"]):
            kv = h * case["kv_heads"] // case["heads"]
            score = (s["km"][where, kv].double() @ s["qm"][:, h].double().T).T.cpu()
            for i in range(case["q_blocks"]):
                rank = torch.sort(score[i], descending=True, stable=True)[1][:room].tolist() if others else []
                found = sorted(always + [others[r] for r in rank])
                out[h, i, :len(found)] = torch.tensor(found, dtype=torch.int32)
        return out.cuda()
    return _exact_attention(case, s)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op in ("prologue", "tables"):
        n = len(_axes(case))
        seq = case["text"] + case["frames"] * case["height"] * case["width"]
        if op == "tables":
            half = case["head_dim"] // 2
            return {"bytes": seq * (4 * n + 8 * half), "flops": 8 * seq * half}
        units = seq * (case["heads"] + case["kv_heads"])
        return {"bytes": units * D * 4 + seq * 4 * n + 8 * D, "flops": units * D * (6 if case["norm"] else 3)}
    if op == "means":
        n = _blocks(case["seq"], case["block"])
        return {"bytes": case["seq"] * case["heads"] * D * 2 + n * (case["heads"] * D * 4 + 4) + 4 * case["seq"] * case["masked"],
                "flops": case["seq"] * case["heads"] * D}
    if op == "select":
        return {"bytes": 4 * D * (case["q_blocks"] * case["heads"] + case["k_blocks"] * case["kv_heads"]) + 4 * case["k_blocks"]
                         + 4 * case["heads"] * case["q_blocks"] * case["topk"],
                "flops": 2 * case["heads"] * case["q_blocks"] * case["k_blocks"] * D}
    keys = min(case["list_len"] * case["k_block"], case["seq_k"]) * (1.0 - 0.5 * case["short"]) * (0.88 if case["masked"] else 1.0)
    nq, nk = _blocks(case["seq_q"], case["q_block"]), _blocks(case["seq_k"], case["k_block"])
    lists = nq * (case["heads"] // case["kv_heads"])                         # lists that share a key head
    named = 1.0 - (1.0 - min(1.0, case["list_len"] / nk)) ** lists          # share of the key blocks that some list names
    return {"bytes": int(4 * case["seq_q"] * case["heads"] * D + 4 * D * case["seq_k"] * case["kv_heads"] * named
                         + 4 * case["heads"] * nq * case["list_len"] + 4 * case["seq_k"] * case["masked"]),
            "flops": int(4 * case["seq_q"] * case["heads"] * keys * D)}
