"""Evaluation loop of the reference's recognition processor (processor/recognition.py:72-76, 110-143)."""
import numpy as np
import torch


def topk_accuracy(result, label, k):
    """Fraction of rows whose label is among the k highest scores (show_topk, recognition.py:72-76)."""
    rank = np.asarray(result).argsort()
    hits = [l in rank[i, -k:] for i, l in enumerate(label)]
    return sum(hits) * 1.0 / len(hits)


def evaluate(model, loader, device, show_topk=(1, 5), evaluation=True, loss_fn=None):
    """model.eval(); run every (data, label) batch of `loader` without gradients; gather the scores.

    Returns dict(result=[n, classes] float array, and with evaluation: label, mean_loss (mean of the per-batch
    mean losses, as the reference reports it) and topk {k: accuracy})."""
    model.eval()
    loss_fn = loss_fn or torch.nn.CrossEntropyLoss()
    losses, results, labels = [], [], []
    for data, label in loader:
        data = data.float().to(device)
        label = label.long().to(device)
        with torch.no_grad():
            output = model(data)
        results.append(output.detach().float().cpu().numpy())
        if evaluation:
            losses.append(loss_fn(output.float(), label).item())
            labels.append(label.cpu().numpy())
    out = {"result": np.concatenate(results)}
    if evaluation:
        out["label"] = np.concatenate(labels)
        out["mean_loss"] = float(np.mean(losses))
        out["topk"] = {k: topk_accuracy(out["result"], out["label"], k) for k in show_topk}
    return out


def _scored(model, loader, device):
    model.eval()
    for data, _ in loader:
        with torch.no_grad():
            yield model(data.float().to(device))


def teacher_targets(model, loader, device, k=16, temperature=2.0):
    """The model's k (or all, if fewer) top logits of every batch of `loader`, in its order: (values [n, k], indices [n, k],
    rest [n]) on the host.  Rows of it, on the device, are the `target` of ddp.Trainer.step at the same temperature."""
    from . import functional as F_
    parts = [F_.top_logits(out, min(k, out.shape[-1]), temperature) for out in _scored(model, loader, device)]
    return F_.TopLogits(*(torch.cat([p[i] for p in parts]).cpu() for i in range(3)))


def pseudo_labels(model, loader, device, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, generator=None):
    """One label per clip of `loader` drawn from the model's scores (functional.sample_labels; temperature 0: the best
    class): dict(label=[n] int64, logp=[n] float32, the log of its share of what was kept).  generator: a CPU
    torch.Generator, drawn from once per clip in the loader's order, whatever the batches are."""
    from . import functional as F_
    parts = []
    for out in _scored(model, loader, device):
        u = torch.rand(out.shape[0], generator=generator).to(out.device)
        parts.append(F_.sample_labels(out, u, temperature, top_k, top_p, min_p))
    return {"label": torch.cat([p[0] for p in parts]).cpu().numpy(), "logp": torch.cat([p[1] for p in parts]).cpu().numpy()}
