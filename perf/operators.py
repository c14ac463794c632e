"""The paged key-value cache and what a serving loop does with it, one operator per case.

``listed()`` holds a dozen calls, from a decoding step of a small batch to long ragged caches; ``draw(rng)`` gives further ones of
the same ranges.  A case is a flat dict; ``op`` says which operator a pass goes through:

  append    new tokens' keys and values into the pages of their sequences
  attend    one new token per sequence against its cache; ``keep`` < 1: over the active blocks of a block mask only; ``weights``: the
            attention weight of every cached key is added up beside it
  weights   the attention weight that the queries of a block-sparse prompt give to every key
  select    which keys of every sequence and kv-head stay: the first, the last, and the heaviest of the rest
  compact   the keys that stay move to the front of their sequence's pages, in place

A cache is (num_pages, page, heads_k, head_dim); lengths are uniform in [len_min, len_max], fixed by ``len_seed``.
With ``own`` false a pass is made of elementary torch operations in 32 bits, with it true of the package's operators.
"""
import numpy as np
import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
SIZES = {"bfloat16": 2, "float16": 2, "float32": 4}


def listed():
    return [
        # a decoding step of a serving batch: one new token per sequence goes into its last page
        dict(name="append_step", op="append", dtype="bfloat16", batch=16, new_min=1, new_max=1, len_min=1024, len_max=4096, len_seed=0,
             heads_k=8, head_dim=64, page=64),
        # prompts of unequal length after their prefill
        dict(name="append_prompts", op="append", dtype="bfloat16", batch=8, new_min=1024, new_max=16384, len_min=0, len_max=0, len_seed=1,
             heads_k=8, head_dim=128, page=128),
        # single precision, as used to check results; a few short sequences, pure call latency
        dict(name="attend_fp32_check", op="attend", dtype="float32", batch=4, len_min=200, len_max=1500, len_seed=2, heads_q=8, heads_k=2,
             head_dim=64, page=16, keep=1.0, k_block=64, weights=False),
        # a long-context batch, small heads, eight queries per key
        dict(name="attend_long", op="attend", dtype="bfloat16", batch=16, len_min=16384, len_max=32768, len_seed=3, heads_q=64, heads_k=8,
             head_dim=64, page=64, keep=1.0, k_block=128, weights=False),
        # a block-sparse step over very long caches
        dict(name="attend_sparse", op="attend", dtype="bfloat16", batch=8, len_min=16384, len_max=65536, len_seed=4, heads_q=32, heads_k=8,
             head_dim=128, page=128, keep=0.3, k_block=128, weights=False),
        # half precision, a head dimension between the tile sizes, small pages, odd lengths, weights kept for a later eviction
        dict(name="attend_fp16_weights", op="attend", dtype="float16", batch=6, len_min=301, len_max=3001, len_seed=5, heads_q=24,
             heads_k=8, head_dim=96, page=16, keep=1.0, k_block=64, weights=True),
        # the prompt's part of the accumulated weight: one layer of a sparse 8k prefill
        dict(name="weights_8k", op="weights", dtype="bfloat16", batch=2, len_min=8192, len_max=8192, len_seed=6, heads_q=16, heads_k=16,
             head_dim=128, q_block=128, k_block=128, causal=True, keep=0.1),
        # ragged GQA samples with small heads and uneven blocks, bidirectional
        dict(name="weights_varlen_gqa", op="weights", dtype="float16", batch=8, len_min=100, len_max=1200, len_seed=7, heads_q=16,
             heads_k=4, head_dim=64, q_block=80, k_block=48, causal=False, keep=0.3),
        # eviction decisions: a small batch, and a long-context one
        dict(name="select_small", op="select", dtype="float32", batch=5, len_min=100, len_max=1000, len_seed=8, heads_k=2, budget=128,
             sink=4, recent=32),
        dict(name="select_long", op="select", dtype="float32", batch=16, len_min=16384, len_max=32768, len_seed=9, heads_k=8, budget=4096,
             sink=16, recent=512),
        # what is kept moves together: small pages and heads, and long caches cut down to an eighth and more
        dict(name="compact_small", op="compact", dtype="float16", batch=4, len_min=200, len_max=1500, len_seed=10, heads_k=2, head_dim=64,
             page=16, budget=128, sink=4, recent=32),
        dict(name="compact_long", op="compact", dtype="bfloat16", batch=8, len_min=8192, len_max=32768, len_seed=11, heads_k=8,
             head_dim=128, page=64, budget=4096, sink=16, recent=512),
    ]


def draw(rng):
    """One more case: sizes over the whole range of the listed ones (log-uniform), odd ones among them."""

    def log_int(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    while True:
        op = rng.choice(["append", "attend", "attend", "attend", "weights", "weights", "select", "compact"])
        dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
        batch = rng.choice([1, 2, 3, 5, 8, 16, 33])
        heads_k = rng.choice([1, 2, 4, 8])
        heads_q = heads_k * rng.choice([1, 2, 3, 4, 8])
        lens = sorted((log_int(1, 32768), log_int(16, 32768)))
        if rng.random() < 0.15:
            lens[0] = 0
        seed = rng.randrange(1 << 30)
        case = dict(op=op, dtype=dtype, batch=batch, len_min=lens[0], len_max=lens[1], len_seed=seed, heads_k=heads_k)
        head_dim, page = rng.choice([32, 64, 64, 80, 96, 128, 128, 256]), rng.choice([16, 32, 48, 64, 128, 256])
        if op == "append":
            new = sorted((log_int(1, 8192), log_int(1, 8192)))
            case.update(new_min=new[0], new_max=new[1], head_dim=head_dim, page=page)
        elif op == "attend":
            case.update(heads_q=heads_q, head_dim=head_dim, page=page, keep=rng.choice([1.0, 1.0, 0.2, 0.5]),
                        k_block=rng.choice([16, 48, 64, 80, 128, 256]), weights=rng.random() < 0.4)
        elif op == "weights":
            lens = sorted((log_int(16, 8192), log_int(16, 8192)))
            case.update(len_min=lens[0], len_max=lens[1], heads_q=heads_q, head_dim=rng.choice([32, 64, 80, 96, 128, 128]),
                        q_block=rng.choice([16, 32, 64, 80, 128]), k_block=rng.choice([16, 48, 64, 80, 128, 256]),
                        causal=rng.random() < 0.7, keep=rng.choice([0.1, 0.2, 0.3, 0.5, 0.7]))
        else:
            budget = log_int(16, 8192)
            sink, recent = rng.choice([0, 1, 4, 16]), rng.choice([0, 1, 7, 64, 512])
            if sink + recent > budget:
                continue
            case.update(budget=budget, sink=sink, recent=recent)
            case.update(dict(head_dim=head_dim, page=page) if op == "compact" else dict(dtype="float32"))
        if op == "weights":
            dear = batch * heads_q * case["len_max"] ** 2 > 2 * 16 * 8192 ** 2 or (dtype == "float32" and work(case)["flops"] > 2e11)
        else:
            dear = batch * heads_k * (case["len_max"] + case.get("new_max", 0)) * case.get("head_dim", 1) * SIZES[dtype] > 1 << 30
        if not dear:
            return case


def _lens(case, what="len"):
    rng = np.random.default_rng(case["len_seed"] + (what == "new"))
    return rng.integers(case[what + "_min"], case[what + "_max"] + 1, size=case["batch"])


def _cu(lens):
    return np.concatenate([[0], np.cumsum(lens)])


def _keep_of(weights, lens, case):
    """Positions that stay, in ascending order and -1 behind them, and how many of them there are: elementary form."""
    n, budget = weights.shape[-1], case["budget"]
    pos = torch.arange(n, device=weights.device)
    length = lens.long()[:, None, None]
    middle = (pos >= case["sink"]) & (pos < length - case["recent"])
    rank = torch.where(middle, weights, torch.inf).masked_fill(pos >= length, -torch.inf)
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    if n < budget:
        best = torch.nn.functional.pad(best, (0, budget - n), value=n)
    best = best[..., :budget]
    best = torch.sort(torch.where(best < length, best, n + 1), dim=-1).values
    return torch.where(best <= n, best, -1).to(torch.int32), lens.clamp(max=budget).to(torch.int32)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype, batch, op = DTYPES[case["dtype"]], case["batch"], case["op"]
    heads_k = case["heads_k"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype)

    lens = _lens(case)
    s = dict(case=case, lens=torch.as_tensor(lens, dtype=torch.int32, device=dev))
    if op == "weights":
        cu = _cu(lens)
        first_q, first_k = _cu(-(-lens // case["q_block"])), _cu(-(-lens // case["k_block"]))
        s["cu"] = torch.as_tensor(cu, dtype=torch.int32, device=dev)
        s["q"] = 2 * normal(int(cu[-1]), case["heads_q"], case["head_dim"])
        s["k"] = normal(int(cu[-1]), heads_k, case["head_dim"])
        mask = torch.rand(heads_k, int(first_q[-1]), int(first_k[-1]), generator=g, device=dev) < case["keep"]
        last = [(np.arange(first_q[b], first_q[b + 1]),
                 first_k[b] + (np.minimum((np.arange(first_q[b + 1] - first_q[b]) + 1) * case["q_block"], lens[b]) - 1) // case["k_block"])
                for b in range(batch)]                       # every row sees itself
        mask[:, torch.as_tensor(np.concatenate([r for r, _ in last]), device=dev), torch.as_tensor(np.concatenate([c for _, c in last]), device=dev)] = True
        s["mask"] = mask
        at, valid = _padded(s)
        s["lse"] = torch.logsumexp(_scores(s, at, valid), dim=-1).permute(0, 2, 1)[valid].contiguous()
        return s
    most = int(lens.max()) + case.get("new_max", 0)
    if op in ("select", "compact") or case.get("weights"):
        size = -(-max(most, 1) // case["page"]) * case["page"] if "page" in case else max(most, 1)
        w = torch.exp(2 * torch.randn(batch, heads_k, size, generator=g, device=dev))
        w = w * (torch.rand(w.shape, generator=g, device=dev) < 0.8)          # keys that no query has looked at
        s["weights"] = w.masked_fill(torch.arange(size, device=dev) >= s["lens"][:, None, None], 0.0)
    if op == "select":
        return s
    page = case["page"]
    pages = -(-(lens + case.get("new_max", 0)) // page)
    width = max(int(pages.max()), 1)
    order = torch.randperm(int(pages.sum()) + 3, generator=g, device=dev).to(torch.int32)
    column = torch.arange(width, device=dev)
    at = torch.as_tensor(_cu(pages)[:-1], device=dev)[:, None] + column
    has = column < torch.as_tensor(pages, device=dev)[:, None]
    s["table"] = torch.where(has, order[at.clamp(max=order.numel() - 1)], 0)
    shape = order.numel(), page, heads_k, case["head_dim"]
    s["k_cache"], s["v_cache"] = normal(*shape), normal(*shape)
    if op == "append":
        cu = _cu(_lens(case, "new"))
        s["cu"] = torch.as_tensor(cu, dtype=torch.int32, device=dev)
        s["k"], s["v"] = (normal(int(cu[-1]), heads_k, case["head_dim"]) for _ in "kv")
    elif op == "attend":
        s["q"] = 2 * normal(batch, case["heads_q"], case["head_dim"])
        s["mask"] = None
        if case["keep"] < 1:
            blocks = -(-width * page // case["k_block"])
            s["mask"] = torch.rand(batch, heads_k, blocks, generator=g, device=dev) < case["keep"]
            newest = (s["lens"].long() - 1).clamp(min=0) // case["k_block"]
            s["mask"].scatter_(2, newest[:, None, None].expand(-1, heads_k, 1), True)
    else:
        s["kept"], s["kept_lens"] = _keep_of(s["weights"], s["lens"], case)
    return s


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        import hbsattn_b200 as hb
        if op == "append":
            lens = hb.append_to_cache(s["k"], s["v"], s["cu"], s["k_cache"], s["v_cache"], s["table"], s["lens"])
            return s["k_cache"], s["v_cache"], lens
        if op == "attend":
            more = dict(block_mask=s["mask"], k_block_size=case["k_block"]) if s["mask"] is not None else {}
            if not case["weights"]:
                return hb.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], **more)
            out = hb.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], key_weights=s["weights"], **more)
            return out, s["weights"]
        if op == "weights":
            return hb.attention_key_weights(s["q"], s["k"], s["lse"], s["cu"], s["cu"], s["mask"], case["q_block"], case["k_block"], case["causal"])
        if op == "select":
            return hb.select_keys(s["weights"], s["lens"], case["budget"], case["sink"], case["recent"])
        hb.compact_cache(s["k_cache"], s["v_cache"], s["table"], s["lens"], s["kept"], s["kept_lens"], key_weights=s["weights"])
        return s["k_cache"], s["v_cache"], s["weights"]
    if op == "append":
        return _append(s)
    if op == "attend":
        return _attend(s)
    if op == "weights":
        return _weights(s)
    if op == "select":
        return _keep_of(s["weights"], s["lens"], case)
    return _compact(s)


def _append(s):
    page = s["case"]["page"]
    cu, token = s["cu"].long(), torch.arange(s["k"].shape[0], device=s["k"].device)
    b = torch.searchsorted(cu[1:], token, right=True)
    pos = s["lens"].long()[b] + token - cu[b]
    at = s["table"].long()[b, pos // page], pos % page
    s["k_cache"][at] = s["k"]
    s["v_cache"][at] = s["v"]
    return s["k_cache"], s["v_cache"], (s["lens"] + cu.diff()).to(torch.int32)


def _attend(s):
    case = s["case"]
    batch, heads_k, d = case["batch"], case["heads_k"], case["head_dim"]
    table = s["table"].long()
    n = table.shape[1] * case["page"]
    k = s["k_cache"][table].reshape(batch, n, heads_k, d).float()
    q = s["q"].float().reshape(batch, heads_k, -1, d)
    x = torch.einsum("bhgd,bnhd->bhgn", q, k) * d ** -0.5
    pos = torch.arange(n, device=q.device)
    seen = (pos < s["lens"][:, None])[:, None, None, :]
    if s["mask"] is not None:
        seen = seen & s["mask"][:, :, pos // case["k_block"]][:, :, None, :]
    x = x.masked_fill(~seen, -torch.inf)
    p = torch.exp(x - x.amax(dim=-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min))
    total = p.sum(dim=-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    v = s["v_cache"][table].reshape(batch, n, heads_k, d).float()
    out = torch.einsum("bhgn,bnhd->bhgd", p, v).reshape(s["q"].shape).to(s["q"].dtype)
    if not case["weights"]:
        return out
    s["weights"] += p.sum(dim=2)
    return out, s["weights"]


def _padded(s):
    """Packed index of every (sample, position), and which of them exist."""
    cu = s["cu"].long()
    pos = torch.arange(s["case"]["len_max"], device=cu.device)
    at, valid = cu[:-1, None] + pos, pos < s["lens"][:, None]
    return torch.where(valid, at, 0), valid


def _scores(s, at, valid):
    """Scaled scores of every sample, padded to the longest one; -inf where a row does not see a key."""
    case, cu = s["case"], s["cu"].long()
    group = case["heads_q"] // case["heads_k"]
    q, k = s["q"][at].float(), s["k"][at].float().repeat_interleave(group, dim=2)
    x = torch.einsum("bihd,bjhd->bhij", q, k) * case["head_dim"] ** -0.5
    pos = torch.arange(at.shape[1], device=at.device)
    lens = cu.diff()
    blocks = [torch.nn.functional.pad((-(-lens // case[n])).cumsum(0), (1, 0))[:-1, None] + pos // case[n] for n in ("q_block", "k_block")]
    i, j = (b.clamp(max=m - 1) for b, m in zip(blocks, s["mask"].shape[1:]))
    seen = s["mask"][:, i[:, :, None], j[:, None, :]].transpose(0, 1).repeat_interleave(group, dim=1)
    seen = seen & (valid[:, :, None] & valid[:, None, :])[:, None]
    if case["causal"]:
        seen &= pos[:, None] >= pos[None, :]
    return x.masked_fill_(~seen, -torch.inf)


def _weights(s):
    at, valid = _padded(s)
    lse = s["lse"][at].transpose(1, 2)[..., None]
    p = torch.exp(_scores(s, at, valid) - torch.where(lse == -torch.inf, torch.inf, lse)).sum(dim=2)
    return p.reshape(p.shape[0], s["case"]["heads_k"], -1, p.shape[-1]).sum(dim=2).transpose(1, 2)[valid]


def _compact(s):
    case, kept = s["case"], s["kept"].long()
    batch, heads_k, budget = kept.shape
    table, page = s["table"].long(), case["page"]
    b, h, j = torch.nonzero(torch.arange(budget, device=kept.device) < s["kept_lens"][:, None, None].expand(-1, heads_k, 1), as_tuple=True)
    src = kept[b, h, j]
    to, of = (table[b, j // page], j % page, h), (table[b, src // page], src % page, h)
    s["k_cache"][to] = s["k_cache"][of]
    s["v_cache"][to] = s["v_cache"][of]
    w = torch.where(torch.arange(s["weights"].shape[-1], device=kept.device) < s["lens"][:, None, None], 0.0, s["weights"])
    w[b, h, j] = s["weights"][b, h, src]
    s["weights"].copy_(w)
    return s["k_cache"], s["v_cache"], s["weights"]


def work(case):
    """Expected over the masks' draw.  Every key that takes part is read once (and written once where it moves), weights are
    read and written, FLOPs are those of the products."""
    size, op = SIZES[case["dtype"]], case["op"]
    lens = _lens(case).astype(np.float64)
    row = case["heads_k"] * case.get("head_dim", 0) * size
    if op == "append":
        return {"bytes": 4.0 * _lens(case, "new").sum() * row + 16.0 * case["batch"], "flops": 0.0}
    if op == "attend":
        newest = np.minimum(lens, (lens - 1) % case["k_block"] + 1)
        keys = float((newest + case["keep"] * (lens - newest)).sum())
        q = case["batch"] * case["heads_q"] * case["head_dim"] * size
        return {"bytes": 2.0 * keys * row + 2.0 * q + (8.0 * keys * case["heads_k"] if case["weights"] else 0.0),
                "flops": 4.0 * keys * case["heads_q"] * case["head_dim"]}
    if op == "weights":
        pairs = 0.0
        for n in lens:
            q0, k0 = np.arange(0, n, case["q_block"]), np.arange(0, n, case["k_block"])
            rows, cols = np.minimum(case["q_block"], n - q0), np.minimum(case["k_block"], n - k0)
            own_block = (q0 + rows - 1) // case["k_block"]
            on = np.where(np.arange(len(k0)) == own_block[:, None], 1.0, case["keep"])
            if case["causal"]:
                on = on * (k0 <= (q0 + rows - 1)[:, None])
            pairs += float(rows @ on @ cols)
        n = lens.sum()
        return {"bytes": n * (row + case["heads_q"] * (case["head_dim"] * size + 4.0) + 4.0 * case["heads_k"]),
                "flops": 2.0 * pairs * case["heads_q"] * case["head_dim"]}
    kept = np.minimum(lens, case["budget"]).sum() * case["heads_k"]
    if op == "select":
        return {"bytes": 4.0 * lens.sum() * case["heads_k"] + 4.0 * case["batch"] * case["heads_k"] * case["budget"], "flops": 0.0}
    moved = (np.minimum(lens, case["budget"]) * (lens > case["budget"])).sum() * case["heads_k"]
    return {"bytes": 4.0 * moved * case["head_dim"] * size + 4.0 * kept + 4.0 * kept + 4.0 * lens.sum() * case["heads_k"], "flops": 0.0}


def exact(case, seed):
    """The definitions, one sequence (and head) at a time, in 64 bits."""
    s, op = prepare(case, seed), case["op"]
    lens = _lens(case)
    if op == "select":
        return None
    if op == "weights":
        d, group = case["head_dim"], case["heads_q"] // case["heads_k"]
        cu, w = _cu(lens), torch.zeros(s["k"].shape[0], case["heads_k"], dtype=torch.float64, device=s["k"].device)
        qb, kb = 0, 0
        for b in range(case["batch"]):
            n = int(lens[b])
            rows = torch.arange(n, device=w.device)
            for h in range(case["heads_q"]):
                q, k = s["q"][cu[b]:cu[b + 1], h].double(), s["k"][cu[b]:cu[b + 1], h // group].double()
                x = (q @ k.T / d ** 0.5 - s["lse"][cu[b]:cu[b + 1], h, None].double()).exp()
                on = s["mask"][h // group][qb + rows[:, None] // case["q_block"], kb + rows[None, :] // case["k_block"]]
                if case["causal"]:
                    on = on.tril()
                w[cu[b]:cu[b + 1], h // group] += torch.where(on, x, 0.0).sum(dim=0)
            qb, kb = qb - (-n // case["q_block"]), kb - (-n // case["k_block"])
        return w
    page = case["page"]

    def slots(b, positions):
        positions = torch.as_tensor(positions, device=s["table"].device)
        return s["table"][b].long()[positions // page], positions % page

    if op == "attend":
        d, group = case["head_dim"], case["heads_q"] // case["heads_k"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
        weights = s["weights"].double() if case["weights"] else None
        for b in range(case["batch"]):
            pos = torch.arange(int(lens[b]), device=out.device)
            for h in range(case["heads_k"]):
                on = pos if s["mask"] is None else pos[s["mask"][b, h, pos // case["k_block"]]]
                if on.numel() == 0:
                    continue
                k, v = (s[c][(*slots(b, on), h)].double() for c in ("k_cache", "v_cache"))
                p = torch.softmax(s["q"][b, h * group:(h + 1) * group].double() @ k.T / d ** 0.5, dim=-1)
                out[b, h * group:(h + 1) * group] = p @ v
                if weights is not None:
                    weights[b, h, on] += p.sum(dim=0)
        return (out, weights) if case["weights"] else out
    caches = [s["k_cache"].clone(), s["v_cache"].clone()]
    if op == "append":
        cu = _cu(_lens(case, "new"))
        for b in range(case["batch"]):
            at = slots(b, np.arange(lens[b], lens[b] + cu[b + 1] - cu[b]))
            for cache, new in zip(caches, (s["k"], s["v"])):
                cache[at] = new[cu[b]:cu[b + 1]]
        return (*(c.double() for c in caches), None)
    weights = s["weights"].clone()
    for b in range(case["batch"]):
        n = int(s["kept_lens"][b])
        weights[b, :, :int(lens[b])] = 0
        for h in range(case["heads_k"]):
            kept = s["kept"][b, h, :n].long()
            for cache, old in zip(caches, (s["k_cache"], s["v_cache"])):
                cache[(*slots(b, np.arange(n)), h)] = old[(*slots(b, kept), h)]
            weights[b, h, :n] = s["weights"][b, h, kept]
    return (*(c.double() for c in caches), weights.double())
