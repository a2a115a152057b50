"""Synthetic data helpers (reference utils/data_loader.py:7-144, utils/loss_funcs.py)."""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F


def generate_model_data(model_name: str, batch_size: int, seq_length: int, vocab_size: int = 32000, image_size: int = 384,
                        device="cpu", seed: int = 0):
    """(inputs, targets) for one batch: token ids for language models, images + class ids for ViT."""
    from ..models import registry

    g = torch.Generator().manual_seed(seed)
    spec = registry.get_spec(model_name)
    if spec.family == "vit":
        x = torch.randn(batch_size, 3, image_size, image_size, generator=g)
        y = torch.randint(0, spec.classes, (batch_size,), generator=g)
    else:
        x = torch.randint(0, vocab_size, (batch_size, seq_length), generator=g)
        y = torch.randint(0, vocab_size, (batch_size, seq_length), generator=g)
    return x.to(device), y.to(device)


def split_microbatches(t: torch.Tensor, microbatch_size: int) -> list[torch.Tensor]:
    return list(t.split(microbatch_size, dim=0))


def split_into(inputs: torch.Tensor, labels: torch.Tensor, microbatches: int):
    """A batch cut into `microbatches` pieces whose sizes differ by at most one sample, larger pieces first
    (reference utils/data_loader.py:54-67, which takes a COUNT where `split_microbatches` above takes a size)."""
    n = len(inputs)
    base, rem = divmod(n, microbatches)
    if base == 0:
        raise ValueError(f"{n} samples cannot fill {microbatches} microbatches")
    sizes = [base + (1 if i < rem else 0) for i in range(microbatches)]
    return inputs.split(sizes), labels.split(sizes)


class RandomTokenDataset(torch.utils.data.Dataset):
    """`size` random token sequences, generated once from `seed`.  `targets`: "next" = the input shifted by one with
    a fresh random last token (language modelling), "random" = independent random tokens, "regression" = one float in
    [0, 1) per position.  Covers the reference's three toy datasets for sequences
    (utils/data_loader.py:70-90, 116-144) and its TensorDataset of random batches (:31-38)."""

    def __init__(self, vocab_size: int, seq_length: int, size: int = 1000, targets: str = "next", seed: int = 0):
        if targets not in ("next", "random", "regression"):
            raise ValueError(f"targets must be next, random or regression, not {targets!r}")
        g = torch.Generator().manual_seed(seed)
        self.inputs = torch.randint(0, vocab_size, (size, seq_length), generator=g)
        if targets == "next":
            self.labels = torch.cat([self.inputs[:, 1:], torch.randint(0, vocab_size, (size, 1), generator=g)], dim=1)
        elif targets == "random":
            self.labels = torch.randint(0, vocab_size, (size, seq_length), generator=g)
        else:
            self.labels = torch.rand(size, seq_length, generator=g)

    def __len__(self) -> int:
        return len(self.inputs)

    def __getitem__(self, i):
        return self.inputs[i], self.labels[i]


class RandomImageDataset(torch.utils.data.Dataset):
    """`size` random images with a class id (`classes` > 0) or a regression target in [0, 1) (`classes` = 0)
    (reference utils/data_loader.py:41-51, 93-113)."""

    def __init__(self, image_size: int, channels: int = 3, size: int = 1000, classes: int = 2, seed: int = 0,
                 dtype: torch.dtype = torch.float32):
        g = torch.Generator().manual_seed(seed)
        self.images = torch.randn(size, channels, image_size, image_size, generator=g).to(dtype)
        self.labels = (torch.randint(0, classes, (size,), generator=g) if classes > 0
                       else torch.rand(size, generator=g).to(dtype))

    def __len__(self) -> int:
        return len(self.images)

    def __getitem__(self, i):
        return self.images[i], self.labels[i]


def get_dataset(model_name: str, *, batch_size: int, batches: int, seq_length: int = 512, vocab_size: int = 32000,
                image_size: int = 224, seed: int = 0) -> torch.utils.data.DataLoader:
    """A loader of `batches` random batches for the model: images for vision models, token ids otherwise
    (reference utils/data_loader.py:24-51 sizes it as warm-up + timed iterations)."""
    from ..models import registry

    if registry.get_spec(model_name).family == "vit":
        ds = RandomImageDataset(image_size, size=batches * batch_size, seed=seed)
    else:
        ds = RandomTokenDataset(vocab_size, seq_length, size=batches * batch_size, targets="random", seed=seed)
    return torch.utils.data.DataLoader(ds, batch_size=batch_size)


def shift_labels(tokens: torch.Tensor, ignore_index: int = -100) -> torch.Tensor:
    """Next-token targets for real text: target[t] = token[t+1], last position ignored."""
    y = torch.full_like(tokens, ignore_index)
    y[..., :-1] = tokens[..., 1:]
    return y


def pack_documents(documents, microbatches: int, B: int, S: int, ignore_index: int = -100, pad: int = 0) -> dict:
    """A batch for `Trainer.train_step_from_host` from token documents (1-D int64 tensors) of any lengths: inputs and targets [M, B, S] and
    "offsets" [M, n + 1].  Documents lie one after another in each microbatch's B S tokens; one that does not fit goes on in the next
    microbatch as a sequence of its own.  Targets are the document's next tokens; the last token of each part and what is left
    over are ignored.  Documents that no microbatch has room for are left out.  Loss and gradients are means over all B S places of a microbatch, as
    they are for batches of equal sequences: ignored ones count as 0, so many short documents and a padded end make both smaller."""
    T = B * S
    x, y = torch.full((microbatches, T), pad, dtype=torch.int64), torch.full((microbatches, T), ignore_index, dtype=torch.int64)
    ends = [[0] for _ in range(microbatches)]
    m = 0
    for doc in documents:
        while doc.numel() and m < microbatches:
            at = ends[m][-1]
            n = min(doc.numel(), T - at)
            x[m, at:at + n] = doc[:n]
            y[m, at:at + n - 1] = doc[1:n]
            ends[m].append(at + n)
            doc = doc[n:]
            m += at + n == T
    width = max(len(e) for e in ends)
    offsets = torch.tensor([e + [e[-1]] * (width - len(e)) for e in ends], dtype=torch.int32)
    return {"inputs": x.view(microbatches, B, S), "targets": y.view(microbatches, B, S), "offsets": offsets}


def random_documents(microbatches: int, B: int, S: int, vocab_size: int, mean: int, generator: torch.Generator) -> dict:
    """A packed batch of random documents whose lengths spread about `mean` (log-normal), at most S tokens each."""
    left, docs = microbatches * B * S, []
    while left > 0:
        n = int(mean * math.exp(0.8 * float(torch.randn((), generator=generator)) - 0.32))
        docs.append(torch.randint(0, vocab_size, (min(max(n, 1), S, left),), generator=generator))
        left -= docs[-1].numel()
    return pack_documents(docs, microbatches, B, S)


class LMLoss(torch.nn.Module):
    def forward(self, logits, targets):
        return F.cross_entropy(logits.flatten(0, -2).float(), targets.flatten())


class RegressionLoss(torch.nn.Module):
    def forward(self, out, targets):
        return F.mse_loss(out.float(), targets.float())
