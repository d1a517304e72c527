"""Cases of the 8-bit integer product family: what is measured, and the operators' plain forms.

Three operators.  With codes(x) = round-half-to-even(127 x / max|x|) of a row (or channel) x and
scale(x) = max|x| / 127:

  matmul   c[m, n] = scale(a_m) scale(w_n) sum_k codes(a_m)[k] codes(w_n)[k]; the weights' codes are made
           once, the activations' within the call
  grouped  the same product where row j of a list sorted by expert meets the weights of its expert;
           "up" takes tokens and sends each to its `top` places, "down" takes sorted rows and puts the
           results back in the order of the assignments; rows of no expert are left as they were
  group    a stable counting sort of assignments by expert: where each expert's rows begin, which
           assignment stands at each place, and the place of each assignment; ids outside the experts
           come last

Sizes are those of the packed products of this repository (4096 x 4096, 4096 x 14336, 4096 x 11008, ...)
and generic ones for experts.
"""
import math

import torch

own = False


# ------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one token through a square projection: the smallest product, where latency counts
        dict(name="matmul f32 1x4096x4096", op="matmul", M=1, K=4096, N=4096, f16=False, strided=False),
        # a small batch of tokens through a wide projection: bound by reading the weights
        dict(name="matmul f32 16x4096x14336", op="matmul", M=16, K=4096, N=14336, f16=False, strided=False),
        # odd in every size, rows inside a wider tensor: a ragged batch between decode and prefill
        dict(name="matmul f16 77x4099x10007", op="matmul", M=77, K=4099, N=10007, f16=True, strided=True),
        # a prompt chunk
        dict(name="matmul f32 512x4096x11008", op="matmul", M=512, K=4096, N=11008, f16=False, strided=False),
        # a long prompt through the projection back to the model's width
        dict(name="matmul f16 2048x14336x4096", op="matmul", M=2048, K=14336, N=4096, f16=True, strided=False),
        # the largest: a batch of prompts
        dict(name="matmul f16 4096x4096x14336", op="matmul", M=4096, K=4096, N=14336, f16=True, strided=False),
        # one token's experts: few rows, each with weights of its own
        dict(name="grouped f32 up 1 of 64", op="grouped", T=1, top=8, E=64, K=2048, N=1024, f16=False, down=False, padded=False),
        # a decode batch with padding, results put back in the tokens' order
        dict(name="grouped f16 down 48 of 64", op="grouped", T=48, top=4, E=64, K=1024, N=2048, f16=True, down=True, padded=True),
        # odd sizes, a few hundred rows over few experts
        dict(name="grouped f32 up 301 of 12", op="grouped", T=301, top=2, E=12, K=1531, N=2777, f16=False, down=False, padded=False),
        # a prompt batch over many experts
        dict(name="grouped f16 up 4096 of 32", op="grouped", T=4096, top=4, E=32, K=2048, N=4096, f16=True, down=False, padded=False),
        # the assignments of a decode batch
        dict(name="group 256 of 64", op="group", R=256, E=64, padded=True),
        # the assignments of a large prompt batch over many experts
        dict(name="group 262144 of 256", op="group", R=262144, E=256, padded=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["matmul", "matmul", "matmul", "grouped", "grouped", "grouped", "group"])
    if op == "matmul":
        while True:
            M, K, N = _log(rng, 1, 4096), _log(rng, 64, 14336), _log(rng, 64, 14336)
            if rng.random() < 0.5:
                K, N = -(-K // 64) * 64, -(-N // 64) * 64
            if M * K * N <= 4096 * 4096 * 14336:
                return dict(op=op, M=M, K=K, N=N, f16=rng.random() < 0.5, strided=rng.random() < 0.3)
    if op == "grouped":
        while True:
            T, E = _log(rng, 1, 4096), _log(rng, 2, 64)
            top, K, N = rng.randint(1, min(8, E)), _log(rng, 64, 4096), _log(rng, 64, 4096)
            if rng.random() < 0.5:
                K, N = -(-K // 64) * 64, -(-N // 64) * 64
            if T * top * K * N <= 4096 * 4 * 2048 * 4096 and E * K * N <= 32 * 2048 * 4096:
                return dict(op=op, T=T, top=top, E=E, K=K, N=N, f16=rng.random() < 0.5, down=rng.random() < 0.5,
                            padded=rng.random() < 0.3)
    return dict(op=op, R=_log(rng, 1, 262144), E=_log(rng, 1, 1024), padded=rng.random() < 0.5)


def work(case):
    if case["op"] == "group":
        # ids in; order, place and the experts' beginnings out, 4 bytes each
        return {"bytes": 4 * (3 * case["R"] + case["E"] + 1), "flops": 0}
    es = 2 if case["f16"] else 4
    if case["op"] == "matmul":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": es * M * K + N * K + 4 * N + es * M * N, "flops": 2 * M * K * N}
    T, top, E, K, N = (case[f] for f in ("T", "top", "E", "K", "N"))
    live = T - T // 8 if case["padded"] else T
    R = live * top
    # experts that hold a row, expected from the routing that _routes draws
    p = _popularity(E)
    touched = sum(1 - (1 - min(1.0, top * q)) ** live for q in p)
    return {"bytes": es * (R if case["down"] else live) * K + touched * N * (K + 4) + 4 * (2 * R + E + 1) + es * R * N,
            "flops": 2 * R * K * N}


# ------------------------------------------------------------------------------------------ the inputs

def _popularity(E):
    """Shares of the experts: some are asked for far more often than others."""
    w = [1.0 / (1 + 0.15 * i) for i in range(E)]
    return [x / sum(w) for x in w]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)


def _activations(rows, K, pitch, dtype, g):
    """Rows of a decoder's stream: normal values, a few channels much larger, rows of different size; the
    last row of a batch is padding."""
    x = torch.randn(rows, pitch, device="cuda", generator=g)
    x *= 1 + 7 * (torch.rand(pitch, device="cuda", generator=g) < 0.005)
    x *= 0.2 + 3 * torch.rand(rows, 1, device="cuda", generator=g)
    if rows > 2:
        x[-1] = 0
    return x.to(dtype)[:, :K]


def _weights(E, K, N, g):
    """f32 weights [E, K, N] with channels of different size."""
    w = torch.randn(E, K, N, device="cuda", generator=g)
    w *= (0.3 + torch.rand(E, 1, N, device="cuda", generator=g)) / math.sqrt(K)
    return w


def _routes(T, top, E, padded, g):
    """`top` different experts for each token, i32 [T, top]; an eighth of a padded batch has none."""
    p = torch.tensor(_popularity(E), device="cuda")
    ids = torch.multinomial(p.expand(T, E), top, generator=g).to(torch.int32)
    if padded and T >= 8:
        ids[T - T // 8:] = -1
    return ids


def _codes64(x, dim):
    """The codes of x along dim, as whole numbers in x's place, and the scale, both held in 64 bits: a value
    next to the border of two codes must not change sides."""
    x = x.double()
    most = x.abs().amax(dim, keepdim=True)
    codes = torch.where(most > 0, torch.round(x * 127 / torch.where(most > 0, most, 1)), 0)
    return codes, most / 127


class State(dict):
    """What the program holds; the framework's handles go with it."""

    def buffer(self, tensor):
        from smith_b200 import device
        span = (tensor.untyped_storage().nbytes() - tensor.storage_offset() * tensor.element_size())
        h = device.wrapDeviceMemory(tensor.data_ptr(), span)
        self.setdefault("handles", []).append(h)
        return h

    def __del__(self):
        for h in self.get("handles", ()):
            from smith_b200 import device
            device.releaseBuffer(h)


def _hold_weights(s, w):
    """The weights as a program keeps them: packed by the framework, or codes and scales."""
    E, K, N = w.shape
    if own:
        from smith_b200 import device
        torch.cuda.synchronize()
        s["packed"] = torch.empty(device.int8PackedBytes(K, N, E), dtype=torch.uint8, device="cuda")
        s["w"] = s.buffer(s["packed"])
        wb = device.wrapDeviceMemory(w.data_ptr(), w.numel() * 4)
        device.int8Pack(device.DTYPE_F32, wb, s["w"], K, N, E)
        device.synchronize()
        device.releaseBuffer(wb)
    else:
        s["codes"] = torch.empty(E, K, N, dtype=torch.int8, device="cuda")
        s["scales"] = torch.empty(E, 1, N, device="cuda")
        for e in range(E):   # one at a time: the 64-bit values of all would not fit beside the rest
            codes, scale = _codes64(w[e], 0)
            s["codes"][e], s["scales"][e] = codes.to(torch.int8), scale.float()


def _sorted_routes(ids, E):
    """The plan of a routed batch: beginnings i32 [E + 1], order and place i32 [R]."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    order = torch.argsort(key, stable=True)
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=order.device)
    counts = torch.zeros(E + 1, dtype=torch.long, device=ids.device).index_add_(0, key, torch.ones_like(key))
    begin = torch.cumsum(counts, 0) - counts
    return begin.to(torch.int32), order.to(torch.int32), place.to(torch.int32)


def _inputs(case, seed):
    """The inputs alone, from the seed."""
    g = _generator(seed)
    if case["op"] == "group":
        R, E = case["R"], case["E"]
        p = torch.tensor(_popularity(E), device="cuda")
        ids = torch.multinomial(p, R, replacement=True, generator=g).to(torch.int32)
        if case["padded"]:
            ids[R - R // 8:] = -1
        return {"ids": ids}
    dtype = torch.float16 if case["f16"] else torch.float32
    if case["op"] == "matmul":
        M, K, N = case["M"], case["K"], case["N"]
        a = _activations(M, K, K + 24 if case["strided"] else K, dtype, g)
        return {"a": a, "weights": _weights(1, K, N, g)}
    T, top, E, K, N = (case[f] for f in ("T", "top", "E", "K", "N"))
    ids = _routes(T, top, E, case["padded"], g)
    a = _activations(T * top if case["down"] else T, K, K, dtype, g)
    return {"a": a, "weights": _weights(E, K, N, g), "ids": ids}


def prepare(case, seed):
    s = State(case=case, **_inputs(case, seed))
    if case["op"] == "group":
        n = case["R"]
        s["begin"] = torch.zeros(case["E"] + 1, dtype=torch.int32, device="cuda")
        s["order"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        s["place"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        names = ("ids", "begin", "order", "place")
    else:
        _hold_weights(s, s.pop("weights"))
        names = ("a", "c")
        if case["op"] == "grouped":
            s["begin"], s["order"], s["place"] = _sorted_routes(s["ids"], case["E"])
            counts = (s["begin"][1:] - s["begin"][:-1]).tolist()
            s["most"], s["rows"] = max(counts), sum(counts)   # of the plan, for the plain form's padding
            names = ("a", "c", "begin", "order", "place")
        rows = case["M"] if case["op"] == "matmul" else case["T"] * case["top"]
        s["c"] = torch.zeros(rows, case["N"], dtype=s["a"].dtype, device="cuda")
    if own:
        torch.cuda.synchronize()
        s["at"] = {n: s.buffer(s[n]) for n in names}
    return s


# ------------------------------------------------------------------------------------------- the calls

def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    if case["op"] == "group":
        return list(_sorted_routes(s["ids"], case["E"]))
    codes, scale = _codes64(s["a"], 1)
    codes, scale = codes.float(), scale.float()
    if case["op"] == "matmul":
        return (codes @ s["codes"][0].float() * scale * s["scales"][0]).to(s["a"].dtype)
    # rows of an expert side by side, padded to the longest: one batched product
    T, top, E, K, N = (case[f] for f in ("T", "top", "E", "K", "N"))
    at = torch.arange(s["rows"], device="cuda")
    order = s["order"][:s["rows"]].long()
    begin = s["begin"].long()
    expert = torch.searchsorted(begin[1:], at, right=True)
    source = at if case["down"] else order // top
    x = torch.zeros(E, s["most"], K, device="cuda")
    x[expert, at - begin[expert]] = codes[source]
    y = torch.bmm(x, s["codes"].float())[expert, at - begin[expert]] * scale[source] * s["scales"][expert, 0]
    c = torch.zeros(T * top, N, dtype=s["a"].dtype, device="cuda")
    c[order if case["down"] else at] = y.to(c.dtype)
    return c


def _run_own(s, case):
    from smith_b200 import device
    at = s["at"]
    if case["op"] == "group":
        device.groupRows(at["ids"], at["begin"], at["order"], at["place"], case["R"], case["E"])
        return [s["begin"], s["order"], s["place"]]
    dtype = device.DTYPE_F16 if case["f16"] else device.DTYPE_F32
    if case["op"] == "matmul":
        device.int8Matmul(dtype, at["a"], s["w"], at["c"], case["M"], case["N"], case["K"], lda=s["a"].stride(0))
    elif case["down"]:
        device.int8MatmulGrouped(dtype, at["a"], s["w"], at["begin"], at["c"], case["T"] * case["top"], case["N"],
                                 case["K"], case["E"], orderBuffer=at["order"])
    else:
        device.int8MatmulGrouped(dtype, at["a"], s["w"], at["begin"], at["c"], case["T"] * case["top"], case["N"],
                                 case["K"], case["E"], positionBuffer=at["place"], fan=case["top"])
    return s["c"]


# ------------------------------------------------------------------------------------ the definition

def exact(case, seed):
    """The definition in 64 bits: round half to even by comparing each value with the middle of its two
    neighbouring codes, products and sums as whole numbers, one expert at a time."""
    i = _inputs(case, seed)
    if case["op"] == "group":
        ids, E = i["ids"].cpu().tolist(), case["E"]
        ids = [e if 0 <= e < E else E for e in ids]
        order = sorted(range(len(ids)), key=lambda r: (ids[r], r))
        place = [0] * len(ids)
        begin = [0] * (E + 1)
        for p, r in enumerate(order):
            place[r] = p
        for e in ids:
            if e < E:
                begin[e + 1] += 1
        for e in range(E):
            begin[e + 1] += begin[e]
        return [torch.tensor(v, dtype=torch.int32) for v in (begin, order, place)]

    def whole(x):   # rows of x
        x = x.double()
        most = x.abs().max(1).values
        safe = torch.where(most > 0, most, torch.ones_like(most)).unsqueeze(1)
        low = torch.floor(127 * x / safe)
        twice = 2 * 127 * x                        # exact: at most 33 significant bits
        middle = (2 * low + 1) * safe              # exact as well
        up = (twice > middle) | ((twice == middle) & (low.remainder(2) == 1))
        return torch.where(most.unsqueeze(1) > 0, low + up.double(), torch.zeros_like(x)), most / 127

    a, sa = whole(i["a"])
    if case["op"] == "matmul":
        w, sw = whole(i["weights"][0].t())
        return (a @ w.t()) * sa.unsqueeze(1) * sw
    top, E = case["top"], case["E"]
    ids = i["ids"].reshape(-1).cpu().long()
    c = torch.zeros(ids.numel(), case["N"], dtype=torch.float64, device="cuda")
    done = 0
    for e in range(E):
        rows = torch.nonzero(ids == e).reshape(-1)
        if rows.numel() == 0:
            continue
        here = torch.arange(done, done + rows.numel())
        source, target = (here, rows) if case["down"] else (rows // top, here)
        w, sw = whole(i["weights"][e].t())
        c[target.cuda()] = (a[source.cuda()] @ w.t()) * sa[source.cuda()].unsqueeze(1) * sw
        done += rows.numel()
    return c
