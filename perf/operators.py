"""Workloads of the operators around the encoder: cross attention to its states (prompt, training and
single-token form), token embeddings with their gradient, and the orthogonalised optimiser step.

`own` selects what `run` calls: the library's entry points (True) or the same mathematics in elementary
torch operations (False)."""
import math

import torch

own = False

NS = (3.4445, -4.7750, 2.0315)  # quintic with steep slope at zero: singular values end in about [0.7, 1.2]
NS_EPS = 1e-7


# ------------------------------------------------------------------------------------------ cases
def _attn(name, B, H, Hkv, Nq, Nk, dh, ragged, train):
    return dict(name=name, op="attention", B=B, H=H, Hkv=Hkv, Nq=Nq, Nk=Nk, dh=dh, ragged=ragged, train=train)


def _embed(name, V, D, B, T, padded, grad):
    return dict(name=name, op="embedding", V=V, D=D, B=B, T=T, padded=padded, grad=grad)


def _ortho(name, rows, cols, batch, muon):
    return dict(name=name, op="orthogonalise", rows=rows, cols=cols, batch=batch, muon=muon)


def listed():
    return [
        # one decoded token per image reads the 197 states of a 224 px / patch 16 encoder: pure latency
        _attn("token_197", 4, 12, 12, 1, 197, 64, False, False),
        # one token over a long shared-head memory (frames of a video, tiles of a large image), ragged batch: HBM bound
        _attn("token_long", 16, 16, 4, 1, 12345, 128, True, False),
        # prompt of a caption over 197 states
        _attn("caption_prompt", 64, 12, 12, 48, 197, 64, False, False),
        # latents that read the states of a large image, odd lengths, padded batch with one entry empty
        _attn("latents_long", 4, 12, 12, 1021, 4099, 64, True, False),
        # training step of a masked decoder: 147 masked tokens read the 50 visible ones, 6 heads
        _attn("masked_decoder_train", 64, 6, 6, 147, 50, 64, False, True),
        # training step of a caption decoder over ragged image features, wide heads shared four to one
        _attn("decoder_train", 8, 16, 4, 509, 1500, 96, True, True),
        # rows of a caption batch for the decoder's input, padded with -1
        _embed("embed_batch", 32000, 768, 64, 256, True, False),
        # gradient of a label table: few tokens, small table
        _embed("embed_grad_small", 1000, 192, 16, 33, False, True),
        # gradient of a caption vocabulary: tokens follow their rank (a few make up most of the batch)
        _embed("embed_grad_batch", 32000, 768, 64, 512, True, True),
        # one square matrix of the smallest configuration (embedding 96)
        _ortho("ortho_96", 96, 96, 1, False),
        # an odd, tall matrix: a head of 257 classes over 1000 features
        _ortho("ortho_tall", 1000, 257, 1, False),
        # optimiser step of the packed q/k/v weights of 12 layers, embedding 768
        _ortho("muon_qkv_768", 768, 2304, 12, True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["token", "prompt", "train", "embed", "embed_grad", "orthogonalise", "muon"])
    limit = {c["name"]: work(c) for c in listed()}
    while True:
        if op in ("token", "prompt", "train"):
            Hkv = rng.choice([1, 2, 3, 4, 6, 8, 12])
            H = Hkv * rng.choice([1, 1, 2, 4])
            case = _attn("", _log_int(rng, 1, 64), H, Hkv, 1 if op == "token" else _log_int(rng, 2, 2048),
                         _log_int(rng, 8, 16384 if op == "token" else 6000), rng.choice([24, 32, 64, 64, 80, 96, 128]),
                         rng.random() < 0.5, op == "train")
            top = limit[dict(token="token_long", prompt="latents_long", train="decoder_train")[op]]
        elif op in ("embed", "embed_grad"):
            case = _embed("", _log_int(rng, 10, 50000), rng.choice([96, 192, 384, 500, 768, 1024]), _log_int(rng, 1, 128),
                          _log_int(rng, 1, 1024), rng.random() < 0.5, op == "embed_grad")
            top = limit["embed_batch" if op == "embed" else "embed_grad_batch"]
        else:
            case = _ortho("", _log_int(rng, 32, 1200), _log_int(rng, 32, 2400), _log_int(rng, 1, 12), op == "muon")
            top = limit["ortho_tall" if op == "orthogonalise" else "muon_qkv_768"]
        w = work(case)
        if w["bytes"] <= top["bytes"] and w["flops"] <= top["flops"]:
            del case["name"]
            return case


def work(case):
    if case["op"] == "attention":
        B, H, Hkv, Nq, Nk, dh = (case[k] for k in ("B", "H", "Hkv", "Nq", "Nk", "dh"))
        # about three quarters of the keys of a ragged batch are there
        keys = Nk if not case["ragged"] else (3 * Nk + 3) // 4
        q, kv = B * Nq * H * dh, B * keys * Hkv * dh
        if case["train"]:  # q, k, v, dout in, out, dq, dk, dv out; 2 products forward, 5 backward
            return dict(bytes=4 * (4 * q + 4 * kv), flops=14 * B * H * Nq * keys * dh)
        return dict(bytes=4 * (2 * q + 2 * kv), flops=4 * B * H * Nq * keys * dh)
    if case["op"] == "embedding":
        n, D, V = case["B"] * case["T"], case["D"], case["V"]
        if case["grad"]:
            return dict(bytes=4 * (n * D + n + V * D), flops=2 * n * D)
        return dict(bytes=4 * (n * D + n + min(n, V) * D), flops=n * D)
    r, n, b = min(case["rows"], case["cols"]), max(case["rows"], case["cols"]), case["batch"]
    # five iterations: x x^T and a a are symmetric (half the products), b x is not
    flops = 5 * b * (r * r * n + r * r * r + 2 * r * r * n)
    return dict(bytes=4 * b * r * n * (5 if case["muon"] else 2), flops=flops)


# ---------------------------------------------------------------------------------------- inputs
def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if case["op"] == "attention":
        B, H, Hkv, Nq, Nk, dh = (case[k] for k in ("B", "H", "Hkv", "Nq", "Nk", "dh"))
        s = dict(q=randn(B, Nq, H, dh), k=randn(B, Nk, Hkv, dh), v=randn(B, Nk, Hkv, dh), scale=dh ** -0.5, lens=None)
        if case["ragged"]:  # lengths from half of the longest up; the last of a larger batch has no states at all
            n = torch.randint((Nk + 1) // 2, Nk + 1, (B,), generator=host)
            n[0] = Nk
            if B >= 4:
                n[-1] = 0
            s["lens"] = n.to(torch.int32).cuda()
        if case["train"]:
            s["dout"] = randn(B, Nq, H, dh) / (B * Nq)  # gradients of a mean loss are small
        return s
    if case["op"] == "embedding":
        V, D, n = case["V"], case["D"], case["B"] * case["T"]
        # frequency falls with the rank: token = V^u - 1
        index = (float(V) ** torch.rand(n, device="cuda", generator=g, dtype=torch.float64)).long() - 1
        index = index.clamp_(0, V - 1)
        if case["padded"]:  # each row of the batch ends in -1 from a length of its own on
            end = torch.randint(case["T"] // 2, case["T"] + 1, (case["B"], 1), generator=host).cuda()
            index[(torch.arange(case["T"], device="cuda")[None, :] >= end).reshape(-1)] = -1
        s = dict(index=index.to(torch.int32), scale=math.sqrt(D))
        if case["grad"]:
            s["dout"] = randn(n, D) / n
        else:
            s["table"] = randn(V, D) * 0.02
        return s
    r, c, b = case["rows"], case["cols"], case["batch"]
    # a gradient of a weight matrix: a few strong directions over a broad floor
    lead = randn(b, r, 8) @ randn(b, 8, c)
    s = dict(g=(0.3 * lead + randn(b, r, c)) * 1e-3)
    if case["muon"]:
        s["m"] = randn(b, r, c) * 5e-3
        s["p"] = randn(b, r, c) * 0.02
        s.update(lr=0.02, momentum=0.95, weight_decay=0.01, update_scale=math.sqrt(max(1.0, r / c)))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        from visiontransformer_amd import vitk
        vitk.init(torch.cuda.current_device())
        s["vitk"] = vitk
        if case["op"] == "attention":
            B, H, Nq, dh = (case[k] for k in ("B", "H", "Nq", "dh"))
            s["out"] = torch.empty_like(s["q"])
            grads = {}
            if case["train"]:
                s["stats"] = torch.empty(B * H, Nq, 2, device="cuda")
                grads = dict(dout=s["dout"], dq=torch.empty_like(s["q"]), dk=torch.empty_like(s["k"]),
                             dv=torch.empty_like(s["v"]))
            s["args"] = vitk.cross_sdpa_args(s["q"], s["k"], s["v"], s["out"], key_len=s["lens"], scale=s["scale"],
                                             stats=s.get("stats"), **grads)
            s["grads"] = grads
        elif case["op"] == "embedding":
            n = case["B"] * case["T"]
            if case["grad"]:
                s["dtable"] = torch.empty(case["V"], case["D"], device="cuda")
                need = vitk.dll().vitk_embedding_bwd_workspace_bytes(n, case["V"], case["D"])
                s["workspace"] = torch.empty((need + 3) // 4, device="cuda")
            else:
                s["out"] = torch.empty(n, case["D"], device="cuda")
        elif case["muon"]:
            s["args"] = vitk.muon_args(s["p"], s["g"], s["m"], lr=s["lr"], momentum=s["momentum"],
                                       weight_decay=s["weight_decay"], update_scale=s["update_scale"], nesterov=True,
                                       steps=5, coefficients=NS, eps=NS_EPS)
        else:
            s["out"] = torch.empty_like(s["g"])
            s["args"] = vitk.newton_schulz_args(s["g"], s["out"], steps=5, coefficients=NS, eps=NS_EPS)
    return s


# ---------------------------------------------------------------------------------- plain forms
def _heads_first(x, group):
    x = x.permute(0, 2, 1, 3)
    if group > 1:
        x = x.repeat_interleave(group, dim=1)
    return x.contiguous()


def _plain_attention(s):
    case = s["case"]
    group = case["H"] // case["Hkv"]
    q, k, v = _heads_first(s["q"], 1), _heads_first(s["k"], group), _heads_first(s["v"], group)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]
    if s["lens"] is not None:
        there = torch.arange(case["Nk"], device="cuda")[None, :] < s["lens"][:, None]
        there = there[:, None, None, :]
        scores = torch.where(there, scores, torch.full_like(scores, -torch.inf))
        m = scores.amax(-1, keepdim=True)
        m = torch.where(torch.isinf(m), torch.zeros_like(m), m)  # no key at all: every exp below is 0
        e = torch.exp(scores - m)
        l = e.sum(-1, keepdim=True)
        p = e / torch.where(l == 0, torch.ones_like(l), l)
    else:
        e = torch.exp(scores - scores.amax(-1, keepdim=True))
        p = e / e.sum(-1, keepdim=True)
    out = torch.matmul(p, v)
    if not case["train"]:
        return out.permute(0, 2, 1, 3).contiguous()
    dout = _heads_first(s["dout"], 1)
    dv = torch.matmul(p.transpose(2, 3).contiguous(), dout)
    dp = torch.matmul(dout, v.transpose(2, 3).contiguous())
    ds = p * (dp - (dout * out).sum(-1, keepdim=True)) * s["scale"]
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q)
    B, Hkv, Nk, dh = case["B"], case["Hkv"], case["Nk"], case["dh"]
    dk, dv = (t.reshape(B, Hkv, group, Nk, dh).sum(2) for t in (dk, dv))
    return [t.permute(0, 2, 1, 3).contiguous() for t in (out, dq, dk, dv)]


def _plain_embedding(s):
    case = s["case"]
    index = s["index"].long()
    there = (index >= 0) & (index < case["V"])
    safe = torch.where(there, index, torch.zeros_like(index))
    if not case["grad"]:
        return s["table"][safe] * (there.float() * s["scale"])[:, None]
    rows = s["dout"] * (there.float() * s["scale"])[:, None]
    return torch.zeros(case["V"], case["D"], device="cuda").index_add_(0, safe, rows)


def _plain_newton_schulz(u):
    a, b, c = NS
    tall = u.shape[1] > u.shape[2]
    x = u.transpose(1, 2).contiguous() if tall else u
    norm = x.double().square().sum((1, 2), keepdim=True).sqrt().float()
    x = x / (norm + NS_EPS)
    for _ in range(5):
        gram = torch.matmul(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return x.transpose(1, 2).contiguous() if tall else x


def _plain_muon(s):
    s["m"].mul_(s["momentum"]).add_(s["g"])
    u = s["g"] + s["momentum"] * s["m"]
    o = _plain_newton_schulz(u)
    s["p"].mul_(1.0 - s["lr"] * s["weight_decay"]).sub_(s["lr"] * s["update_scale"] * o)
    return [s["p"], s["m"]]


# ------------------------------------------------------------------------------------------- run
def run(s):
    case = s["case"]
    if not own:
        if case["op"] == "attention":
            return _plain_attention(s)
        if case["op"] == "embedding":
            return _plain_embedding(s)
        return _plain_muon(s) if case["muon"] else _plain_newton_schulz(s["g"])
    vitk = s["vitk"]
    if case["op"] == "attention":
        vitk.cross_sdpa_fwd(s["args"])
        if not case["train"]:
            return s["out"]
        vitk.cross_sdpa_bwd(s["args"])
        return [s["out"], s["grads"]["dq"], s["grads"]["dk"], s["grads"]["dv"]]
    if case["op"] == "embedding":
        if not case["grad"]:
            vitk.embedding_fwd(s["table"], s["index"], s["out"], scale=s["scale"])
            return s["out"]
        vitk.embedding_bwd(s["dout"], s["index"], s["dtable"], scale=s["scale"], workspace=s["workspace"])
        return s["dtable"]
    if case["muon"]:
        vitk.muon(s["args"])
        return [s["p"], s["m"]]
    vitk.newton_schulz(s["args"])
    return s["out"]


# ------------------------------------------------------------------------------------- 64 bits
def _exact_attention(case, s):
    B, H, Hkv, Nk, train = case["B"], case["H"], case["Hkv"], case["Nk"], case["train"]
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    lens = [Nk] * B if s["lens"] is None else s["lens"].tolist()
    for b in range(B):
        n = lens[b]
        if n == 0:
            continue
        for h in range(H):
            j = h // (H // Hkv)
            kk, vv, qq = k[b, :n, j].contiguous(), v[b, :n, j].contiguous(), q[b, :, h].contiguous()
            p = torch.softmax(torch.mm(qq, kk.t().contiguous()) * s["scale"], dim=1)
            out[b, :, h] = torch.mm(p, vv)
            if train:
                do = s["dout"][b, :, h].double().contiguous()
                dp = torch.mm(do, vv.t().contiguous())
                ds = s["scale"] * p * (dp - (p * dp).sum(1, keepdim=True))
                dq[b, :, h] = torch.mm(ds, kk)
                dk[b, :n, j] += torch.mm(ds.t().contiguous(), qq)
                dv[b, :n, j] += torch.mm(p.t().contiguous(), do)
    return [out, dq, dk, dv] if train else out


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    if case["op"] == "embedding":
        kept = (s["index"] >= 0).nonzero()[:, 0]
        token = s["index"][kept].long()
        if case["grad"]:
            order = torch.argsort(token, stable=True)
            total = torch.zeros(case["V"], case["D"], device="cuda", dtype=torch.float64)
            total.index_put_((token[order],), s["dout"][kept[order]].double(), accumulate=True)
            return total * s["scale"]
        out = torch.zeros(case["B"] * case["T"], case["D"], device="cuda", dtype=torch.float64)
        out[kept] = s["table"].double()[token] * s["scale"]
        return out
    g = s["g"].double()
    if case["muon"]:
        m = s["momentum"] * s["m"].double() + g
        g = g + s["momentum"] * m
    res = torch.empty_like(g)
    for i in range(case["batch"]):
        x = g[i] / (torch.linalg.norm(g[i]) + NS_EPS)
        for _ in range(5):  # x p(x^T x) or p(x x^T) x, whichever matrix is the smaller one
            if x.shape[0] <= x.shape[1]:
                w = torch.mm(x, x.t().contiguous())
                x = NS[0] * x + NS[1] * torch.mm(w, x) + NS[2] * torch.mm(w, torch.mm(w, x))
            else:
                w = torch.mm(x.t().contiguous(), x)
                x = NS[0] * x + NS[1] * torch.mm(x, w) + NS[2] * torch.mm(torch.mm(x, w), w)
        res[i] = x
    if case["muon"]:
        p = s["p"].double()
        return [p - s["lr"] * s["weight_decay"] * p - s["lr"] * s["update_scale"] * res, m]
    return res
