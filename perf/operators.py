"""The operators of answering with a policy next to training it: keys and values written to a paged cache (bf16, or e4m3
with a scale per token and head) and read back, attention of new tokens over that cache, and the verification of drafted
tokens.  Each case is one call as a serving loop makes it.

Heads, head dimensions and vocabularies are those of the policies this package is timed on (12/2, 28/4, 40/8 and 64/8 heads
of 128, 14/2 heads of 64; vocabularies of 1000, 32000 and about 152k), prompts and answers those of its packed samples."""
import math
import os
import random
import sys

import torch

own = False

_HEADS = ((12, 2, 128), (28, 4, 128), (40, 8, 128), (64, 8, 128), (14, 2, 64))
FP8 = torch.float8_e4m3fn
FP8_MAX, FP8_FLOOR = 448.0, 1e-30


# ------------------------------------------------------------------------------------------------ the list
def listed():
    return [
        # one new token of each of 64 sequences into one layer's cache: the smallest write, where the launch is what counts
        _cache("write_tokens", kind="write", B=64, q=(1, 1), k=(128, 1024), Hkv=4, D=128, page=16, fp8=False),
        # the keys and values of a full budget of prompts, quantised as they are written
        _cache("write_prompts_fp8", kind="write", B=56, q=(128, 1024), k=(128, 1024), Hkv=8, D=128, page=64, fp8=True),
        # what a quantised cache holds of a batch of answers, back in packed form (to hand it to another layer of storage)
        _cache("read_answers_fp8", kind="read", B=40, q=(1, 1), k=(256, 2048), Hkv=4, D=128, page=16, fp8=True),
        # the same of a small batch of a 0.5B-class policy, plain
        _cache("read_small_d64", kind="read", B=13, q=(1, 1), k=(100, 777), Hkv=2, D=64, page=32, fp8=False),
        # one token of four short answers: the smallest attention call
        _attn("attn_token_few", B=4, q=(1, 1), k=(128, 1024), Hq=12, Hkv=2, D=128, page=16, fp8=False),
        # one token of each of 128 answers of ragged lengths, a 7B-class policy: all of it is reading the cache
        _attn("attn_token_batch", B=128, q=(1, 1), k=(128, 8192), Hq=28, Hkv=4, D=128, page=64, fp8=False),
        # the same on long contexts and a quantised cache, a 70B-class policy
        _attn("attn_token_long_fp8", B=48, q=(1, 1), k=(1024, 32768), Hq=64, Hkv=8, D=128, page=16, fp8=True),
        # one to eight drafted tokens a sequence, a 0.5B-class policy
        _attn("attn_drafts_d64", B=32, q=(1, 8), k=(128, 4096), Hq=14, Hkv=2, D=64, page=32, fp8=False),
        # the answers of one prompt scored over the prompt's pages, which they share
        _attn("attn_group_scored", B=8, q=(256, 1024), k=(2048, 3000), Hq=12, Hkv=2, D=128, page=16, fp8=False, shared=1500),
        # a piece of a long prompt over what came before it, quantised, a 32B-class policy: the largest call
        _attn("attn_piece_long_fp8", B=1, q=(4096, 4096), k=(32768, 32768), Hq=40, Hkv=8, D=128, page=64, fp8=True),
        # drafts looked up in the prompt (no distribution of their own), a small vocabulary in bf16
        dict(kind="verify", name="verify_lookup", B=4, q_lo=2, q_hi=5, V=32000, fp32=False, draft=False, lens=1),
        # drafts of a smaller model, a full batch
        dict(kind="verify", name="verify_batch", B=64, q_lo=1, q_hi=9, V=151936, fp32=True, draft=True, lens=2),
    ]


def _cache(name, kind, B, q, k, Hkv, D, page, fp8):
    return dict(kind=kind, name=name, B=B, q_lo=q[0], q_hi=q[1], k_lo=k[0], k_hi=k[1], Hkv=Hkv, D=D, page=page, fp8=fp8, lens=len(name))


def _attn(name, B, q, k, Hq, Hkv, D, page, fp8, shared=0):
    return dict(kind="attn", name=name, B=B, q_lo=q[0], q_hi=q[1], k_lo=k[0], k_hi=k[1], Hq=Hq, Hkv=Hkv, D=D, page=page, fp8=fp8,
                shared=shared, lens=len(name))


def draw(rng):
    """Another case of the same ranges: batch sizes, lengths and pages spread over them, over their logarithm where they are wide."""
    def near(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))
    kind = rng.choice(["write", "read", "attn", "attn", "attn", "verify"])
    if kind == "verify":
        lo = rng.randint(1, 3)
        return dict(kind=kind, B=near(1, 64), q_lo=lo, q_hi=lo + rng.randint(0, 6), V=rng.choice([1000, 32000, 128256, 151936, near(1000, 152064)]),
                    fp32=rng.random() < 0.6, draft=rng.random() < 0.7, lens=rng.randrange(1 << 20))
    Hq, Hkv, D = rng.choice(_HEADS)
    case = dict(kind=kind, Hkv=Hkv, D=D, page=rng.choice([16, 32, 64, 128, 256]), fp8=rng.random() < 0.5, lens=rng.randrange(1 << 20))
    if kind != "attn":
        new = rng.random() < 0.4
        case["B"] = near(1, 128) if new else near(1, 40)
        case["k_lo"] = near(16, 256)
        case["k_hi"] = case["k_lo"] + near(1, 1024)
        case["q_lo"], case["q_hi"] = (1, 1) if new else (case["k_lo"], case["k_hi"])
        return case
    case["Hq"], case["shared"] = Hq, 0
    form = rng.choice(["token", "token", "drafts", "chunk"])
    case["B"] = near(1, 128 if form == "token" else 64 if form == "drafts" else 8)
    case["q_lo"], case["q_hi"] = {"token": (1, 1), "drafts": (1, rng.randint(2, 9)), "chunk": (near(16, 256), near(256, 2048))}[form]
    case["k_lo"] = near(64, 2048)
    case["k_hi"] = case["k_lo"] + near(64, 6000)
    if form == "chunk" and rng.random() < 0.5:
        case["shared"] = case["k_lo"] // 2
    return case


# ------------------------------------------------------------------------------------------------ sizes of a case
def _lens(case):
    """(new tokens, keys with them) of every sequence."""
    rng = random.Random(case["lens"])
    q = [rng.randint(case["q_lo"], case["q_hi"]) for _ in range(case["B"])]
    if case["kind"] == "verify":
        return q, q
    k = [max(rng.randint(case["k_lo"], case["k_hi"]), n) for n in q]
    if case["kind"] == "write" and case["q_hi"] > 1:      # whole prompts
        k = list(q)
    shared = case.get("shared", 0)
    return q, [max(n, m + shared) for n, m in zip(k, q)]


def work(case):
    q, k = _lens(case)
    if case["kind"] == "verify":
        rows = (2 if case["draft"] else 1) * case["B"]
        return {"bytes": rows * case["V"] * (4 if case["fp32"] else 2) + 40 * sum(q), "flops": 2 * rows * case["V"]}
    row = case["Hkv"] * case["D"]
    held = 2 * (row + 4 * case["Hkv"]) if case["fp8"] else 4 * row           # one token's keys and values in the cache
    if case["kind"] != "attn":
        n = sum(q if case["kind"] == "write" else k)
        return {"bytes": n * (4 * row + held), "flops": 2 * n * row}
    shared = case["shared"] // case["page"] * case["page"]
    keys = sum(k) - (case["B"] - 1) * shared
    pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(q, k))
    return {"bytes": keys * held + 4 * sum(q) * case["Hq"] * case["D"], "flops": 4 * case["D"] * case["Hq"] * pairs}


# ------------------------------------------------------------------------------------------------ inputs
def _offsets(n, dev):
    return torch.tensor([0] + torch.tensor(n).cumsum(0).tolist(), dtype=torch.int32, device=dev)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(dev).manual_seed(seed)
    q, k = _lens(case)
    st = dict(case=case, T=sum(q), keys=sum(k), max_q=max(q), max_k=max(k), cu_q=_offsets(q, dev), cu_k=_offsets(k, dev),
              lens=torch.tensor(k, dtype=torch.int32, device=dev))
    if case["kind"] == "verify":
        return _prepare_verify(st, case, g, dev)
    page, Hkv, D = case["page"], case["Hkv"], case["D"]
    # every sequence has pages of its own, in no order, but for those of a shared prompt
    same = case.get("shared", 0) // page
    need = [(n + page - 1) // page - same for n in k]
    pages = sum(need) + same
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    width = max(need) + same
    table = torch.full((case["B"], width), -1, dtype=torch.int32)
    host, at = order.cpu(), same
    for b, n in enumerate(need):
        table[b, :same] = host[:same]
        table[b, same:same + n] = host[at:at + n]
        at += n
    st["table"] = table.to(dev)
    new = lambda n, h: torch.randn(n, h, D, generator=g, device=dev).bfloat16()      # noqa: E731
    shape = (pages, page, Hkv, D)
    if case["kind"] == "write":
        st["k"], st["v"] = new(st["T"], Hkv), new(st["T"], Hkv)
        for n in ("k_cache", "v_cache"):
            st[n] = torch.zeros(shape, dtype=FP8 if case["fp8"] else torch.bfloat16, device=dev)
            st[n[0] + "_scale"] = torch.zeros(shape[:3], device=dev) if case["fp8"] else None
        return st
    for n in ("k", "v"):
        x = new(pages * page, Hkv)
        code, scale = _quantised(x) if case["fp8"] else (x, None)
        st[n + "_cache"], st[n + "_scale"] = code.view(shape), None if scale is None else scale.view(shape[:3])
    if case["kind"] == "attn":
        st["q"] = new(st["T"], case["Hq"])
    return st


def _prepare_verify(st, case, g, dev):
    T, B, V = st["T"], case["B"], case["V"]
    dtype = torch.float32 if case["fp32"] else torch.bfloat16
    logits = 2.5 * torch.randn(T, V, generator=g, device=dev)
    first, last = (torch.zeros(T, dtype=torch.bool, device=dev) for _ in range(2))
    first[st["cu_q"][:-1].long()] = True
    last[st["cu_q"][1:].long() - 1] = True
    ids = torch.randint(0, V, (T,), generator=g, device=dev)
    st["draft"] = None
    if case["draft"]:                    # a smaller model's distribution, near the policy's, and tokens drawn from it
        smaller = logits[~last] + 0.7 * torch.randn(T - B, V, generator=g, device=dev)
        st["draft"] = smaller.softmax(-1).to(dtype)
        if T > B:
            noise = -torch.log(-torch.log(torch.rand(T - B, V, generator=g, device=dev).clamp_(1e-9, 1 - 1e-7)))
            ids[~first] = (smaller + noise).argmax(-1)
    else:                                # text that was copied: the policy likes it, or not at all
        t = torch.arange(T, device=dev)[~last]
        logits[t, ids[t + 1]] += 18.0 * (torch.rand(T - B, generator=g, device=dev) < 0.7)
    st["target"], st["ids"] = logits.softmax(-1).to(dtype), ids
    st["u"] = torch.rand(T, generator=g, device=dev)
    return st


# ------------------------------------------------------------------------------------------------ the pass
def run(st):
    kind = st["case"]["kind"]
    if own:
        return _own(st, kind)
    return {"write": _plain_write, "read": _plain_read, "attn": _plain_attention, "verify": _plain_verify}[kind](st)


def _own(st, kind):
    package = os.path.join(os.getcwd(), "async-grpo-nccl_amd")     # the directory name is not an importable package name
    if package not in sys.path:
        sys.path.insert(0, package)
    from fgrpo import ops
    if kind == "verify":
        accepted, tokens = ops.verify_drafts(st["target"], st["draft"], st["ids"], st["u"], st["cu_q"])
        return {"accepted": accepted, "tokens": tokens}
    cache = ops.PagedCache(st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"])
    if kind == "write":
        ops.paged_cache_write(cache, st["k"], st["v"], st["table"], st["lens"], st["cu_q"])
        return {"k": cache.k, "v": cache.v, "k_scale": cache.k_scale, "v_scale": cache.v_scale}
    if kind == "read":
        k, v = ops.paged_cache_read(cache, st["table"], st["lens"], st["cu_k"], st["keys"])
        return {"k": k, "v": v}
    out, lse = ops.paged_attention(st["q"], cache, st["table"], st["lens"], st["cu_q"], max_len=st["max_q"], return_lse=True)
    return {"out": out, "lse": lse}


def _quantised(x):
    """(codes, scale) of the rows of x: the largest finite magnitude of a row becomes 448."""
    x = x.float()
    top = x.abs().nan_to_num(0.0, 0.0, 0.0).amax(-1).clamp(min=FP8_FLOOR)
    most = torch.full_like(top, FP8_MAX)           # number / tensor would be the number times a rounded reciprocal
    return (x * (most / top).unsqueeze(-1)).to(FP8), top / most


def _places(cu, n):
    """The sequence of each of n packed rows, and the row's place in it."""
    t = torch.arange(n, device=cu.device)
    b = torch.searchsorted(cu, t, right=True, out_int32=True).long() - 1
    return b, t - cu[b]


def _slots(st, b, at):
    page = st["case"]["page"]
    return st["table"][b, at // page].long() * page + at % page


def _plain_write(st):
    b, i = _places(st["cu_q"], st["T"])
    n = st["cu_q"][b + 1] - st["cu_q"][b]
    slot = _slots(st, b, st["lens"][b].long() - n + i)
    _put(st, "k", slot)
    _put(st, "v", slot)
    return {"k": st["k_cache"], "v": st["v_cache"], "k_scale": st["k_scale"], "v_scale": st["v_scale"]}


def _put(st, name, slot):
    cache, scale, x = st[name + "_cache"], st[name + "_scale"], st[name]
    if scale is None:
        cache.view(-1, *cache.shape[2:])[slot] = x
    else:
        code, s = _quantised(x)
        cache.view(torch.uint8).view(-1, *cache.shape[2:])[slot] = code.view(torch.uint8)
        scale.view(-1, scale.shape[2])[slot] = s


def _held(st, name, slot):
    """The cached rows of these slots in 32 bits."""
    cache, scale = st[name + "_cache"], st[name + "_scale"]
    if scale is None:
        return cache.view(-1, *cache.shape[2:])[slot].float()
    x = cache.view(torch.uint8).view(-1, *cache.shape[2:])[slot].view(FP8).float()
    return x.mul_(scale.view(-1, scale.shape[2])[slot].unsqueeze(-1))


def _plain_read(st):
    b, i = _places(st["cu_k"], st["keys"])
    slot = _slots(st, b, i)
    return {"k": _held(st, "k", slot).bfloat16(), "v": _held(st, "v", slot).bfloat16()}


def _plain_attention(st):
    case = st["case"]
    B, Hq, Hkv, D, mq, mk = case["B"], case["Hq"], case["Hkv"], case["D"], st["max_q"], st["max_k"]
    G, dev = Hq // Hkv, st["q"].device
    lens, cu = st["lens"].long(), st["cu_q"].long()
    n = cu[1:] - cu[:-1]
    i, j = torch.arange(mq, device=dev), torch.arange(mk, device=dev)
    q = st["q"][(cu[:-1, None] + i).clamp(max=st["T"] - 1)].float()                           # [B, mq, Hq, D]
    q = q.view(B, mq, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * mq, D)
    slot = _slots(st, torch.arange(B, device=dev)[:, None], j.expand(B, mk).minimum(lens[:, None] - 1))
    k, v = (_held(st, x, slot).permute(0, 2, 1, 3).contiguous() for x in ("k", "v"))          # [B, Hkv, mk, D]
    s = torch.matmul(q, k.transpose(2, 3)).mul_(D ** -0.5).view(B, Hkv, G, mq, mk)
    seen = (j < lens[:, None, None]) & (j <= (lens - n)[:, None, None] + i[:, None])          # [B, mq, mk]
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(top).exp_()
    total = s.sum(-1, keepdim=True)
    out = torch.matmul(s.view(B, Hkv, G * mq, mk), v).view(B, Hkv, G, mq, D).div_(total)
    b, i = _places(st["cu_q"], st["T"])
    lse = (top + total.log()).squeeze(-1)
    return {"out": out.permute(0, 3, 1, 2, 4)[b, i].reshape(st["T"], Hq, D).bfloat16(),
            "lse": lse.permute(0, 3, 1, 2)[b, i].reshape(st["T"], Hq).t().contiguous()}


def _plain_verify(st):
    target, draft, ids, u = st["target"], st["draft"], st["ids"], st["u"]
    T, B, dev = st["T"], st["case"]["B"], target.device
    cu = st["cu_q"].long()
    drafts = cu[1:] - cu[:-1] - 1
    i = torch.arange(st["max_q"], device=dev)
    t = (cu[:-1, None] + i).clamp(max=T - 1)                         # [B, max_q] rows of the target
    d = ids[(t + 1).clamp(max=T - 1)]
    at = torch.arange(B, device=dev)
    p_d = target[t, d].double()
    if draft is None or draft.shape[0] == 0:
        q_d = torch.ones_like(p_d)
    else:
        q_d = draft[(t - at[:, None]).clamp(max=T - B - 1), d].double()
    kept = (u[t].double() * q_d < p_d) & (i < drafts[:, None])
    accepted = kept.int().cumprod(1).sum(1)                          # up to the first that is not
    row = cu[:-1] + accepted
    p = target[row].double().clamp(min=0)
    refused = accepted < drafts
    if draft is None or draft.shape[0] == 0:
        gone = torch.zeros_like(p)
        gone[at, ids[(row + 1).clamp(max=T - 1)]] = 1.0
    else:
        gone = draft[(row - at).clamp(max=T - B - 1)].double()
    rest = torch.where(refused[:, None], (p - gone).clamp(min=0), p)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, p)
    sums = rest.cumsum(1)
    last = (rest.shape[1] - 1) - (rest > 0).flip(1).int().argmax(1)
    token = (sums <= u[row].double()[:, None] * sums[:, -1:]).sum(1).minimum(last)
    b, place = _places(st["cu_q"], T)
    tokens = torch.where(place < accepted[b], ids[(torch.arange(T, device=dev) + 1).clamp(max=T - 1)], -1)
    tokens = torch.where(place == accepted[b], token[b], tokens)
    return {"accepted": accepted.to(torch.int32), "tokens": tokens}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _exact_verify(st):
    target, draft, ids, u, cu = st["target"], st["draft"], st["ids"].tolist(), st["u"].double().tolist(), st["cu_q"].tolist()
    accepted, tokens = [], [-1] * st["T"]
    for b, (lo, hi) in enumerate(zip(cu, cu[1:])):
        n = 0
        while lo + n + 1 < hi:
            d = ids[lo + n + 1]
            q = 1.0 if draft is None else float(draft[lo - b + n, d])
            if not u[lo + n] * q < float(target[lo + n, d]):
                break
            tokens[lo + n] = d
            n += 1
        p = target[lo + n].double()
        if lo + n + 1 < hi:
            gone = torch.nn.functional.one_hot(st["ids"][lo + n + 1], p.numel()).double() if draft is None else draft[lo - b + n].double()
            rest = torch.relu(p - gone)
            p = rest if float(rest.sum()) > 0 else p
        sums = p.cpu().cumsum(0)
        tokens[lo + n] = min(int(torch.searchsorted(sums, u[lo + n] * float(sums[-1]), right=True)), int(p.nonzero()[-1]))
        accepted.append(n)
    return {"accepted": torch.tensor(accepted, dtype=torch.int32), "tokens": torch.tensor(tokens)}


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "verify":
        return _exact_verify(st)
    q, k = _lens(case)
    page = case["page"]
    table, out = st["table"].tolist(), {}
    rows = lambda b, lo, hi: torch.tensor([table[b][j // page] * page + j % page for j in range(lo, hi)], device=st["table"].device)   # noqa: E731

    def double(name, slot):
        c, s = st[name + "_cache"], st[name + "_scale"]
        flat = c.double().view(-1, case["Hkv"], case["D"])[slot]
        return flat if s is None else flat * s.double().view(-1, case["Hkv"])[slot][..., None]

    if case["kind"] == "write":
        slot = torch.cat([rows(b, k[b] - q[b], k[b]) for b in range(case["B"])])
        for name in ("k", "v"):
            x = st[name].double()
            held = torch.zeros(st[name + "_cache"].shape, dtype=torch.float64, device=x.device)
            scale = None
            if case["fp8"]:
                scale = torch.zeros(held.shape[:3], dtype=torch.float64, device=x.device)
                s = x.abs().amax(-1).clamp(min=FP8_FLOOR) / 448
                scale.view(-1, case["Hkv"])[slot] = s
                x = x / s[..., None]
            held.view(-1, case["Hkv"], case["D"])[slot] = x
            out[name], out[name + "_scale"] = held, scale
        return out
    if case["kind"] == "read":
        return {n: double(n, torch.cat([rows(b, 0, k[b]) for b in range(case["B"])])) for n in ("k", "v")}
    G, D = case["Hq"] // case["Hkv"], case["D"]
    cached = {n: None for n in ("k", "v")}
    o = torch.empty(st["T"], case["Hq"], D, dtype=torch.float64, device=st["q"].device)
    lse = torch.empty(case["Hq"], st["T"], dtype=torch.float64, device=o.device)
    first = 0
    for b in range(case["B"]):
        slot = rows(b, 0, k[b])
        for n in cached:
            c, s = st[n + "_cache"].view(-1, case["Hkv"], D), st[n + "_scale"]
            x = (c.view(torch.uint8)[slot].view(FP8) if s is not None else c[slot]).double()
            cached[n] = x if s is None else x * s.view(-1, case["Hkv"])[slot].double()[..., None]
        at = torch.arange(k[b] - q[b], k[b], device=o.device)
        hidden = torch.arange(k[b], device=o.device)[None, :] > at[:, None]
        for h in range(case["Hq"]):
            s = st["q"][first:first + q[b], h].double() @ cached["k"][:, h // G].T / math.sqrt(D)
            s = s.masked_fill(hidden, -math.inf)
            lse[h, first:first + q[b]] = torch.logsumexp(s, 1)
            o[first:first + q[b], h] = torch.softmax(s, 1) @ cached["v"][:, h // G]
        first += q[b]
    return {"out": o, "lse": lse}
