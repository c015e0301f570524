"""`PagedLM`: a `CausalLM` served from a paged cache: sequences that come and go, each with its own length.

`CausalLM` keeps one contiguous cache per batch and one length for all of its rows, as the reference does. Here a call takes any
new tokens of any open sequences, a decode step's single tokens and chunks of prompts together: their rows go through
the model's own products, norms and embedding one after another, and `paged.append` and `paged.attention` place and read keys
and values sequence by sequence. Pages are taken as sequences grow and given back when they are closed.

Keys and values are float32, bfloat16 (half the memory and traffic of a decode step) or "int4" (4.5 bits a word, a seventh of them: see `paged`
for how a word is rounded). Either way the attention's sums run in an order of the kernels' own choice, so logits agree with `CausalLM`'s to rounding, not
to the bit, and in 4 bits to what is left of its keys and values.
"""
import numpy as np
import torch

from .. import _native, paged
from ..transformer import NORM_KINDS, _stream, _vp, add, add_norm, norm

CACHES = {"bfloat16": torch.bfloat16, "float32": torch.float32, "int4": "int4"}


def _integers(x):
    if x.dtype.kind not in "iu":
        raise TypeError("token ids must be integers")
    return x.astype(np.int32)


class PagedLM(object):
    def __init__(self, lm, n_pages, *, page=64, cache="bfloat16"):
        """`lm`: a CausalLM on one device. `n_pages` pages of `page` positions for each of its layers."""
        if lm.world != 1:
            raise ValueError("a paged cache serves a model on one device, got one cut over %d" % lm.world)
        if cache not in CACHES:
            raise ValueError("cache must be one of %s, got %r" % (", ".join(sorted(CACHES)), cache))
        cfg = lm.config
        self.lm = lm
        self.cache = paged.PagedCache(n_pages, cfg.n_kv_heads, cfg.head_dim, page=page, layers=cfg.n_layers, dtype=CACHES[cache], device=lm.device)
        self.positions = min([cfg.max_positions] + [blk.ceiling for blk in lm.blocks])  # as far as the contiguous model goes
        self.cos = self.sin = None
        if lm.blocks and lm.blocks[0].rope and self.positions:  # of every position: a row takes its own
            self.cos, self.sin = lm.blocks[0].rope_tables(0, self.positions)

    def open(self):
        """A new, empty sequence: its name for `feed` and `close`."""
        return self.cache.open()

    def close(self, sequence):
        self.cache.close(sequence)

    def length(self, sequence):
        return self.cache.length[sequence]

    def feed(self, sequences, ids):
        """New tokens ids[i] (each at least one) of sequences[i]: logits (len(sequences), vocab) on the device, of each one's last.
        A call that fails leaves the sequences as they were."""
        lm = self.lm
        sequences = list(sequences)
        ids = [np.asarray(x).reshape(-1) for x in ids]
        counts = [x.size for x in ids]
        if len(ids) != len(sequences) or not ids or min(counts) < 1:
            raise ValueError("feed takes at least one token for each sequence")
        longest = max(self.cache.length[s] + n for s, n in zip(sequences, counts))
        if longest > self.positions:
            raise ValueError("absolute position %d is at or beyond max_positions %d" % (longest - 1, self.positions))
        if lm.pos_table is not None and longest > lm.pos_table.shape[0]:
            raise ValueError("position table of %d rows is too short" % lm.pos_table.shape[0])
        ids = [_integers(x) for x in ids]
        before = [self.cache.length[s] for s in sequences]
        tables = self.cache.extend(sequences, counts)
        try:
            return self._forward(ids, counts, before, longest, *tables)
        except BaseException:  # the tokens were not (all) written: they do not count
            self.cache.retract(sequences, counts)
            raise

    def _forward(self, ids, counts, before, longest, table, cu, lengths):
        lm, cfg, dev = self.lm, self.lm.config, self.lm.device
        total, st = sum(counts), _stream(dev)
        host = np.concatenate(ids + [np.arange(p, p + n, dtype=np.int32) for p, n in zip(before, counts)] + [np.cumsum(counts) - 1]).astype(np.int32)
        words = torch.from_numpy(host).pin_memory().to(dev, non_blocking=True)

        def rows_of(weight, at):
            out = torch.empty((total, cfg.d_model), dtype=torch.float32, device=dev)
            _native.call("b200i_embedding", dev.index, st, _vp(out), _vp(weight), _vp(at), total, weight.shape[0], cfg.d_model, _vp(lm._status))
            return out

        x, delta = rows_of(lm.embed, words[:total]), None
        if lm.pos_table is not None:
            x = add(x, rows_of(lm.pos_table, words[total:2 * total].contiguous()))
        for i, blk in enumerate(lm.blocks):
            x, delta = blk.forward_rows(x, delta, self.cache.k[i], self.cache.v[i], table, cu, lengths, self.cos, self.sin, max(counts), longest)
        last = words[2 * total:].long()  # only each sequence's last row goes through the final norm and the head
        x = x.index_select(0, last)
        if delta is None:
            h = norm(x, lm.final_w, lm.final_b, cfg.norm_eps, NORM_KINDS[cfg.norm])
        else:
            h = add_norm(x, delta.index_select(0, last), lm.final_w, lm.final_b, cfg.norm_eps, NORM_KINDS[cfg.norm])[1]
        return lm.head(h)

    def generate(self, prompts, max_new_tokens, chunk=512):
        """Greedy continuations of prompts of any lengths: a list of int32 arrays, prompt and continuation. Prompts are fed `chunk` tokens
        at a time, and sequences whose prompt is through go on one token a call beside them."""
        prompts = [np.asarray(p).reshape(-1) for p in prompts]
        if not prompts or min(p.size for p in prompts) < 1:
            raise ValueError("a prompt has at least one token")
        prompts = [_integers(p) for p in prompts]
        names = [self.open() for _ in prompts]
        try:
            out = [list(p) for p in prompts]
            goal = [p.size + int(max_new_tokens) for p in prompts]
            while True:
                # the last token of a sequence is not fed: nothing would be asked of it
                live = [i for i, n in enumerate(names) if len(out[i]) < goal[i]]
                if not live:
                    break
                parts = [np.asarray(out[i][self.length(names[i]):][:int(chunk)], dtype=np.int32) for i in live]
                logits = self.feed([names[i] for i in live], parts)
                best = self.lm.argmax_device(logits).cpu().numpy()
                for i, token in zip(live, best):
                    if self.length(names[i]) == len(out[i]):  # all that is known of it has been fed
                        out[i].append(int(token))
            self.lm.check_ids()
            self.lm.check_status()
            return [np.asarray(x, dtype=np.int32) for x in out]
        finally:
            for n in names:
                self.close(n)
