"""Cases of the operators around one shared network that many requests use: the forward pass with a low-rank adapter per
request, the gradients of those adapters, the clipping of gradients by their global norm, and the controls on logits
(priors, candidate masks, penalties) with their softmax.

Each case is computed in a plain form (elementary torch operations) or, where `own` is set, by streamz_amd's entry points.
All data is f32, the type of every matrix of the library; losses and squared sums are added in 64 bits."""
import math

import numpy as np
import torch

own = False

FEATURES = 60   # values of one window


def listed():
    net = {"h1": 512, "h2": 256, "out": 16}
    wide = {"h1": 2048, "h2": 2048, "out": 256}
    return [
        # one window of one live stream: nothing but latency
        dict(name="forward one window", op="forward", rows=1, requests=1, slots=4, rank=8, mixed=False, controls=False, **net),
        # a step of 64 live streams, one window each, every stream with an adapter and a candidate list of its own
        dict(name="forward 64 streams", op="forward", rows=64, requests=64, slots=64, rank=16, mixed=False, controls=True, **net),
        # ten minutes of audio in 32 ragged clips, 24 adapters, a candidate list for each clip
        dict(name="forward 32 clips", op="forward", rows=66140, requests=32, slots=24, rank=16, mixed=False, controls=True, **net),
        # four minutes in 8 clips through the wide network
        dict(name="forward wide", op="forward", rows=26456, requests=8, slots=8, rank=32, mixed=False, controls=False, **wide),
        # adapting to one five-second enrolment clip
        dict(name="train one clip", op="train", rows=550, requests=1, slots=2, rank=8, mixed=False, controls=False, **net),
        # one optimiser step of 16 adapters over ten minutes whose windows come shuffled
        dict(name="train 16 adapters", op="train", rows=66140, requests=16, slots=16, rank=16, mixed=True, controls=True, **net),
        # the same for the wide network, two minutes
        dict(name="train wide", op="train", rows=13228, requests=8, slots=8, rank=32, mixed=False, controls=False, **wide),
        # the gradient of one network, six tensors, between the sum over ranks and the update
        dict(name="clip one network", op="clip", nets=1, groups=1, **net),
        # eight wide networks trained together under one norm: 48 tensors
        dict(name="clip eight wide networks", op="clip", nets=8, groups=1, **wide),
        # the windows of a one-minute clip, one candidate list
        dict(name="controls one clip", op="controls", rows=6614, classes=16, sets=1, penalties=False, probs=True),
        # 100 one-minute clips, 64 speakers, running counts of each clip
        dict(name="controls 100 clips", op="controls", rows=661400, classes=64, sets=100, penalties=True, probs=True),
        # a large register of speakers, every row with counts and candidates of its own
        dict(name="controls large register", op="controls", rows=1024, classes=50001, sets=1024, penalties=True, probs=True),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["forward", "forward", "train", "train", "clip", "controls"])
    if op == "clip":
        case = {"op": op, "nets": _spread(rng, 1, 40), "h1": _spread(rng, 32, 2048), "h2": _spread(rng, 16, 2048), "out": _spread(rng, 2, 256)}
        while case["nets"] * (61 * case["h1"] + (case["h1"] + 1) * case["h2"]) > 36_000_000:
            case["nets"] = max(1, case["nets"] // 2)
        case["groups"] = rng.choice([1, case["nets"]])
        return case
    if op == "controls":
        classes = _spread(rng, 2, 60000)
        rows = _spread(rng, 1, min(600_000, 40_000_000 // classes))
        return {"op": op, "rows": rows, "classes": classes, "sets": _spread(rng, 1, max(1, min(rows, 40_000_000 // classes))), "penalties": rng.random() < 0.5,
                "probs": rng.random() < 0.7}
    h1, h2 = (rng.choice([(512, 256), (2048, 2048), (1024, 768)]) if rng.random() < 0.5 else (_spread(rng, 24, 1500), _spread(rng, 16, 1500)))
    out = _spread(rng, 2, 256)
    most = min(60_000, int(1.5e11 / (h1 * (h2 + FEATURES) + h2 * out)))
    rows, rank = _spread(rng, 1, most if op == "forward" else max(2, most // 2)), _spread(rng, 1, 64)
    slots = _spread(rng, 1, max(1, min(200, 4096 // rank, 200_000_000 // (rows * rank))))
    return {"op": op, "rows": rows, "requests": _spread(rng, 1, min(rows, 300)), "slots": slots, "rank": rank, "mixed": rng.random() < 0.3,
            "controls": rng.random() < 0.5, "h1": h1, "h2": h2, "out": out}


def _net_shapes(c):
    return [(FEATURES, c["h1"]), (c["h1"],), (c["h1"], c["h2"]), (c["h2"],), (c["h2"], c["out"]), (c["out"],)]


def _adapter_shapes(c):
    r = c["rank"]
    return [(c["h1"], r), (r, c["h2"]), (c["h2"], r), (r, c["out"])]


def _split(flat, shapes):
    """Views of one flat vector (or of each row of a matrix of them) in the given shapes."""
    out, at = [], 0
    for s in shapes:
        n = math.prod(s)
        out.append(flat[..., at:at + n].reshape(flat.shape[:-1] + tuple(s)))
        at += n
    return out


class _View:
    """Device memory that the library owns, as torch takes it in; the tensor keeps its owner."""

    def __init__(self, ptr, shape, owner, typestr="<f4"):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "data": (ptr, False), "version": 2}


def _make_controls(g, dev, sets, classes, penalties, rows):
    c = {"sets": sets}
    c["bias"] = torch.randn(sets, classes, generator=g, device=dev)
    words = (classes + 31) // 32
    share = torch.randint(1, 4, (sets, 1, 1), generator=g, device=dev)   # a quarter, half or three quarters of the classes
    bits = (torch.randint(0, 4, (sets, words, 32), generator=g, device=dev) < share).to(torch.int64)
    if sets >= 8:
        bits[sets // 2] = 0   # a request none of whose candidates this network knows
    bits[0] = 1
    c["allow"] = (bits << torch.arange(32, device=dev)).sum(-1).to(torch.uint32 if hasattr(torch, "uint32") else torch.int64)
    c["set_of_row"] = torch.sort(torch.randint(0, sets, (rows,), generator=g, device=dev, dtype=torch.int32)).values
    if penalties:
        seen = torch.randint(0, 40, (sets, classes), generator=g, device=dev, dtype=torch.int32)
        c["counts"] = (seen - 30).clamp(min=0)
        c["repetition"] = 1.0 + torch.rand(sets, generator=g, device=dev)
        c["presence"] = torch.rand(sets, generator=g, device=dev) - 0.5   # below zero: who has spoken is likely to go on
        c["frequency"] = 0.1 * torch.rand(sets, generator=g, device=dev)
    return c


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = {"case": case}
    uniform = lambda shape, a: (2 * torch.rand(shape, generator=g, device=dev) - 1) * a  # noqa: E731
    if case["op"] == "clip":
        shapes = _net_shapes(case) * case["nets"]
        s["grads"] = [torch.randn(math.prod(x), generator=g, device=dev) * 10.0 for x in shapes]
        s["live"] = torch.full((case["groups"],), 6614.0, device=dev)
        # half of the norm that such gradients have: the clipping happens
        s["max_norm"] = 0.5 * 10.0 / 6614.0 * math.sqrt(sum(x.numel() for x in s["grads"]) / case["groups"])
        s["group"] = [i // 6 if case["groups"] > 1 else 0 for i in range(len(shapes))]
        s["group_dev"] = torch.tensor(s["group"], device=dev)
        if own:
            import streamz_amd
            s["out"] = [torch.empty_like(x) for x in s["grads"]]
            s["norms"] = torch.empty(case["groups"], device=dev)
            s["clip"] = streamz_amd.GradClip([(x.data_ptr(), x.numel()) for x in s["grads"]], outputs=[x.data_ptr() for x in s["out"]],
                                             groups=s["group"], live=s["live"].data_ptr())
        return s
    if case["op"] == "controls":
        s["logits"] = 3.0 * torch.randn(case["rows"], case["classes"], generator=g, device=dev)
        s["controls"] = _make_controls(g, dev, case["sets"], case["classes"], case["penalties"], case["rows"])
        if own:
            import streamz_amd
            s["handle"] = streamz_amd.LogitControls(**{k: v if k == "sets" else v.data_ptr() for k, v in s["controls"].items()})
        return s
    # forward and train: a trained network's weights, features as the extractor's z-scores, one slot for each request
    flat = [uniform(x, (math.sqrt(3.0 / x[0]) if i % 2 == 0 else 0.1)) for i, x in enumerate(_net_shapes(case))]
    s["params"] = torch.cat([x.reshape(-1) for x in flat])
    P = sum(math.prod(x) for x in _adapter_shapes(case))
    a2, b2, a3, b3 = _adapter_shapes(case)
    part = [uniform((case["slots"],) + x, math.sqrt(3.0 / k)) for x, k in ((a2, case["h1"]), (b2, 8 * case["rank"]), (a3, case["h2"]), (b3, 8 * case["rank"]))]
    s["adapters"] = torch.cat([x.reshape(case["slots"], -1) for x in part], dim=1).contiguous()
    assert s["adapters"].shape[1] == P
    s["scale"] = 0.5
    n, q = case["rows"], case["requests"]
    cuts = torch.sort(torch.randint(0, n + 1, (q - 1,), generator=g, device=dev)).values
    request = torch.bucketize(torch.arange(n, device=dev), cuts, right=True) if n != q else torch.arange(n, device=dev)
    if case["mixed"]:
        request = request[torch.randperm(n, generator=g, device=dev)]
    slot_of = torch.randint(0, case["slots"], (q,), generator=g, device=dev) if q != case["slots"] else torch.randperm(q, generator=g, device=dev)
    if q >= 8:
        slot_of[q // 3] = -1   # a request without an adapter
    s["slots"] = slot_of[request].to(torch.int32)
    s["x"] = torch.randn(n, FEATURES, generator=g, device=dev)
    if n >= 100:
        s["x"][torch.randint(0, n, (n // 100,), generator=g, device=dev)] = 0.0   # windows without signal
    s["labels"] = torch.randint(0, case["out"], (n,), generator=g, device=dev, dtype=torch.int32)
    s["controls"] = None
    if case["controls"]:
        s["controls"] = _make_controls(g, dev, q, case["out"], False, n)
        s["controls"]["set_of_row"] = request.to(torch.int32)
    if own:
        import streamz_amd
        s["net"] = streamz_amd.SimpleNeuralNet(FEATURES, case["h1"], case["h2"], case["out"], init=s["params"].cpu().numpy())
        s["bank"] = streamz_amd.Adapters(s["net"], case["slots"], case["rank"], scale=s["scale"], init=s["adapters"].cpu().numpy())
        s["bank"].reserve(n, training=case["op"] == "train")
        s["handle"] = streamz_amd.LogitControls(**{k: v if k == "sets" else v.data_ptr() for k, v in s["controls"].items()}) if s["controls"] else None
        if case["op"] == "train":
            grad = torch.as_tensor(_View(s["bank"].grad_ptr(), (s["bank"].grad_len(),), s["bank"]), device=dev)
            s["grad"] = grad[:case["slots"] * P].view(case["slots"], P)
            s["stats"] = grad[case["slots"] * P:].view(case["slots"], 2)
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------

def _allowed(c, classes, index):
    """Truth values [rows][classes] of the candidate mask."""
    words = c["allow"].to(torch.int64)[index]
    bit = torch.arange(classes, device=words.device)
    return (words[:, bit // 32] >> (bit % 32)) & 1 > 0


def _controlled(logits, c):
    """(controlled logits, probabilities); without controls the logits and their softmax."""
    z = logits
    if c is not None:
        index = c["set_of_row"].to(torch.int64)
        if "counts" in c:
            n = c["counts"][index].float()
            rep = c["repetition"][index][:, None]
            z = torch.where(n > 0, torch.where(z > 0, z / rep, z * rep) - c["presence"][index][:, None], z)
            z = z - c["frequency"][index][:, None] * n
        z = z + c["bias"][index]
        z = torch.where(_allowed(c, z.shape[1], index), z, torch.full_like(z, -math.inf))
    top = z.max(dim=1, keepdim=True).values
    e = torch.exp(z - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(dim=1, keepdim=True)
    return z, torch.where(total > 0, e / total, torch.zeros_like(e))


def _low(x, a, slots, scale):
    """scale x A[slot] of every row, laid out [rows][slots * rank] with zeros at the other slots."""
    k, r = a.shape[1], a.shape[2]
    every = (x @ a.permute(1, 0, 2).reshape(k, -1)).view(x.shape[0], -1, r) * scale
    mine = slots[:, None] == torch.arange(a.shape[0], device=x.device)
    return torch.where(mine[:, :, None], every, torch.zeros_like(every)).view(x.shape[0], -1)


def _layers(s):
    case = s["case"]
    w1, b1, w2, b2, w3, b3 = _split(s["params"], _net_shapes(case))
    A2, B2, A3, B3 = _split(s["adapters"], _adapter_shapes(case))
    h1 = torch.clamp(s["x"] @ w1 + b1, min=0.0)
    u2 = _low(h1, A2, s["slots"], s["scale"])
    h2 = torch.tanh(h1 @ w2 + b2 + u2 @ B2.reshape(-1, case["h2"]))
    u3 = _low(h2, A3, s["slots"], s["scale"])
    return h1, u2, h2, u3, h2 @ w3 + b3 + u3 @ B3.reshape(-1, case["out"])


def _plain_train(s):
    case, S, r = s["case"], s["case"]["slots"], s["case"]["rank"]
    w3 = _split(s["params"], _net_shapes(case))[4]
    A2, B2, A3, B3 = _split(s["adapters"], _adapter_shapes(case))
    h1, u2, h2, u3, logits = _layers(s)
    _, p = _controlled(logits, s["controls"])
    label = s["labels"].to(torch.int64)
    t = (label[:, None] == torch.arange(case["out"], device=label.device)).float()
    live = (s["x"] != 0).any(dim=1) & (s["slots"] >= 0)
    if s["controls"] is not None:
        live = live & (_allowed(s["controls"], case["out"], s["controls"]["set_of_row"].to(torch.int64)) & (t > 0)).any(dim=1)
    d3 = torch.where(live[:, None], p - t, torch.zeros_like(p))
    loss = torch.where(live, -torch.log(torch.clamp((p * t).sum(dim=1), min=1e-12)), torch.zeros_like(p[:, 0]))
    g3 = _low(d3, B3.transpose(1, 2), s["slots"], s["scale"])
    d2 = (d3 @ w3.t() + g3 @ A3.transpose(1, 2).reshape(-1, case["h2"])) * (1.0 - h2 * h2)
    g2 = _low(d2, B2.transpose(1, 2), s["slots"], s["scale"])
    parts = [(h1.t() @ g2).view(-1, S, r).permute(1, 0, 2), (u2.t() @ d2).view(S, r, -1),
             (h2.t() @ g3).view(-1, S, r).permute(1, 0, 2), (u3.t() @ d3).view(S, r, -1)]
    mine = (s["slots"][:, None] == torch.arange(S, device=label.device)).double()
    stats = torch.stack([mine.t() @ loss.double(), mine.t() @ live.double()], dim=1).float()
    return {"grad": torch.cat([x.reshape(S, -1) for x in parts], dim=1), "stats": stats}


def _plain_clip(s):
    squares = torch.stack([x.double().square().sum() for x in s["grads"]])
    norm = torch.zeros(s["case"]["groups"], dtype=torch.float64, device=squares.device).index_add_(0, s["group_dev"], squares).sqrt() / s["live"].double()
    factor = torch.where(norm > s["max_norm"], s["max_norm"] / norm, torch.ones_like(norm)).float()[s["group_dev"]]
    return {"grads": _as_one([x * f for x, f in zip(s["grads"], factor)]), "norms": norm.float()}


def _as_one(tensors):
    """At most 48 outputs: with more tensors, the first 47 and the others end to end."""
    return tensors if len(tensors) <= 48 else tensors[:47] + [torch.cat(tensors[47:])]


def run(s):
    case = s["case"]
    if own:
        return _run_own(s, torch.cuda.current_stream().cuda_stream)
    if case["op"] == "clip":
        return _plain_clip(s)
    if case["op"] == "controls":
        return _controlled(s["logits"], s["controls"])[1 if case["probs"] else 0]
    if case["op"] == "train":
        return _plain_train(s)
    logits = _layers(s)[4]
    return {"logits": logits, "probs": _controlled(logits, s["controls"])[1]}


# ---- the framework's calls ---------------------------------------------------------------------------------

def _run_own(s, stream):
    case = s["case"]
    if case["op"] == "clip":
        s["clip"].run(s["max_norm"], norms_ptr=s["norms"].data_ptr(), stream=stream)
        return {"grads": _as_one(s["out"]), "norms": s["norms"]}
    if case["op"] == "controls":
        import streamz_amd
        out = torch.empty_like(s["logits"])
        streamz_amd.control_logits_dev(s["logits"].data_ptr(), case["rows"], case["classes"], s["handle"], out.data_ptr(),
                                       probs=case["probs"], stream=stream)
        return out
    if case["op"] == "train":
        s["bank"].zero_grad_dev(stream)
        s["bank"].accumulate_dev(s["net"], s["x"].data_ptr(), s["labels"].data_ptr(), s["slots"].data_ptr(), case["rows"], controls=s["handle"],
                                 stream=stream)
        return {"grad": s["grad"], "stats": s["stats"]}
    logits = torch.empty(case["rows"], case["out"], device="cuda")
    probs = torch.empty_like(logits)
    s["net"].forward_adapted_dev(s["bank"], s["x"].data_ptr(), s["slots"].data_ptr(), case["rows"], logits_ptr=logits.data_ptr(),
                                 probs_ptr=probs.data_ptr(), controls=s["handle"], stream=stream)
    return {"logits": logits, "probs": probs}


# ---- in 64 bits --------------------------------------------------------------------------------------------

def _exact_controls(logits, c):
    """Controlled logits and probabilities, a set at a time, with the masks unpacked by numpy."""
    z = logits.clone()
    if c is not None:
        rows, classes = z.shape
        bits = np.unpackbits(np.ascontiguousarray(c["allow"].to(torch.int64).cpu().numpy().astype("<u4")).view(np.uint8), axis=1, bitorder="little")
        allowed = torch.from_numpy(bits[:, :classes].astype(bool)).to(z.device)
        which = c["set_of_row"].cpu().numpy()
        order = np.argsort(which, kind="stable")
        for part in np.split(order, np.flatnonzero(np.diff(which[order])) + 1):
            k, at = int(which[part[0]]), torch.from_numpy(part).to(z.device)
            v = z[at]
            if "counts" in c:
                n = c["counts"][k].double()
                seen = n > 0
                v[:, seen] = torch.where(v[:, seen] > 0, v[:, seen] / c["repetition"][k].double(), v[:, seen] * c["repetition"][k].double()) - c["presence"][k].double()
                v = v - n * c["frequency"][k].double()
            v = v + c["bias"][k].double()
            v[:, ~allowed[k]] = -math.inf
            z[at] = v
    empty = torch.isinf(z).all(dim=1)
    p = torch.softmax(z, dim=1)
    p[empty] = 0.0
    return z, p


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        total = [math.fsum(float(torch.linalg.vector_norm(x.double())) ** 2 for x, k in zip(s["grads"], s["group"]) if k == group) for group in range(case["groups"])]
        norms = [math.sqrt(t) / float(s["live"][k]) for k, t in enumerate(total)]
        return {"grads": _as_one([x.double() * min(1.0, s["max_norm"] / norms[k]) for x, k in zip(s["grads"], s["group"])]),
                "norms": torch.tensor(norms, dtype=torch.float64, device="cuda")}
    if case["op"] == "controls":
        return _exact_controls(s["logits"].double(), s["controls"])[1 if case["probs"] else 0]
    # the layers row group by row group of each slot, the gradients by differentiating the loss
    w1, b1, w2, b2, w3, b3 = [x.double() for x in _split(s["params"], _net_shapes(case))]
    bank = s["adapters"].double().requires_grad_(case["op"] == "train")
    slots = s["slots"].cpu().numpy()
    logits = torch.empty(case["rows"], case["out"], dtype=torch.float64, device="cuda")
    stats = torch.zeros(case["slots"], 2, dtype=torch.float64, device="cuda")
    for k in np.unique(slots):
        at = torch.from_numpy(np.flatnonzero(slots == k)).cuda()
        x = s["x"][at].double()
        h1 = torch.relu(torch.addmm(b1, x, w1))
        z = torch.addmm(b2, h1, w2)
        a2, c2, a3, c3 = _split(bank[int(k)], _adapter_shapes(case)) if k >= 0 else (None,) * 4
        h2 = torch.tanh(z if k < 0 else z + s["scale"] * ((h1 @ a2) @ c2))
        l = torch.addmm(b3, h2, w3) if k < 0 else torch.addmm(b3, h2, w3) + s["scale"] * ((h2 @ a3) @ c3)
        logits[at] = l.detach()
        if case["op"] != "train" or k < 0:
            continue
        label = s["labels"][at].to(torch.int64)
        shift, count = torch.zeros_like(l), (x.abs().sum(dim=1) > 0)
        if s["controls"] is not None:   # a prior moves logits, a mask takes classes out: both as an added constant
            part = {**s["controls"], "set_of_row": s["controls"]["set_of_row"][at]}
            shift = _exact_controls(torch.zeros_like(l), part)[0]
            count = count & torch.isfinite(shift.gather(1, label[:, None])[:, 0])
        if bool(count.any()):
            lp = torch.log_softmax((l + shift)[count], dim=1).gather(1, label[count][:, None])[:, 0]
            # below 1e-12 the reported loss stops, its gradient does not
            stats[int(k), 0] = -torch.clamp(lp.detach(), min=math.log(1e-12)).sum()
            stats[int(k), 1] = count.sum()
            (-lp.sum()).backward()
    if case["op"] == "train":
        return {"grad": bank.grad if bank.grad is not None else torch.zeros_like(bank), "stats": stats}
    return {"logits": logits, "probs": _exact_controls(logits, s["controls"])[1]}


# ---- what a pass cannot do without -------------------------------------------------------------------------

def work(case):
    if case["op"] == "clip":
        n = case["nets"] * sum(math.prod(x) for x in _net_shapes(case))
        return {"bytes": 8 * n, "flops": 3 * n}
    if case["op"] == "controls":
        n, table = case["rows"] * case["classes"], case["sets"] * case["classes"]
        return {"bytes": 8 * n + table * (8 if case["penalties"] else 4) + table // 8 + 4 * case["rows"], "flops": 12 * n}
    n, r, h1, h2, out = case["rows"], case["rank"], case["h1"], case["h2"], case["out"]
    used = min(case["slots"], case["requests"])
    net, bank = sum(math.prod(x) for x in _net_shapes(case)), used * sum(math.prod(x) for x in _adapter_shapes(case))
    flops = 2 * n * (FEATURES * h1 + h1 * h2 + h2 * out) + 2 * n * r * (h1 + 2 * h2 + out)
    if case["op"] == "forward":
        return {"bytes": 4 * (n * FEATURES + n + net + bank + 2 * n * out), "flops": flops}
    # the loss, the products back to the first adapted layer, and the factors' gradients
    flops += 2 * n * h2 * out + 2 * n * r * (2 * out + 2 * h2 + 2 * h2 + h1)
    return {"bytes": 4 * (n * FEATURES + 2 * n + net + 2 * bank), "flops": flops}
